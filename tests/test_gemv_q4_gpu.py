"""4-bit Linear on up to eight rows against the formula in 64 bits: every type of x and of the scales, every group, reductions that end
inside a word, a group and a block, rows of weights that end inside a tile, pitches, epilogues, what lies behind a row."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.gpu

UNIT = {K.THB_F32: 2.0 ** -24, K.THB_F16: 2.0 ** -11, K.THB_BF16: 2.0 ** -8}
TORCH = {K.THB_F32: torch.float32, K.THB_F16: torch.float16, K.THB_BF16: torch.bfloat16}
E4M3 = "e4m3"


@pytest.fixture(scope="module")
def lib():
    return K.load()


def up(v, m):
    return (v + m - 1) // m * m


class Layer:
    def __init__(self, dtype, n, k, m, group, zeros=True, x8=False, sdtype=K.THB_F16, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed + 100003 * m + k)
        self.dtype, self.n, self.k, self.m, self.group, self.x8 = dtype, n, k, m, group, x8
        groups = (k + group - 1) // group
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        # codes and scales in their pitches; what lies behind a row is anything
        self.w = torch.randint(0, 256, (m, up((k + 1) // 2, 16) + 16), device="cuda", generator=g, dtype=torch.uint8)
        self.s = (torch.exp(rand(m, groups + 1)) * 0.05).to(TORCH[sdtype])
        self.z = torch.randint(0, 16, (m, groups + 3), device="cuda", generator=g, dtype=torch.uint8) if zeros else None
        x = rand(n, up(k, 16) + 16)
        self.x_scale = torch.exp(rand(n)).contiguous() if x8 else None
        self.x = x.to(torch.float8_e4m3fn) if x8 else x.to(TORCH[dtype])
        self.x[:, k:] = float("nan")
        al = K.ALIGN[dtype]
        self.y = torch.full((n, up(m, al) + al), 7.0, device="cuda", dtype=TORCH[dtype])
        d = self.d = K.GemvQ4Desc(dtype=dtype, N=n, K=k, M=m, group=group, x_ld=self.x.stride(0), y_ld=self.y.stride(0),
                                  w_ld=self.w.stride(0), s_ld=self.s.stride(0), wscale_dtype=sdtype, w=self.w.data_ptr(),
                                  wscale=self.s.data_ptr())
        if zeros:
            d.wzero, d.z_ld = self.z.data_ptr(), self.z.stride(0)

    def call(self, lib, stream=None):
        return lib.thb_gemv_q4_fwd(C.byref(self.d), self.x.data_ptr(), self.x_scale.data_ptr() if self.x8 else None, self.y.data_ptr(), stream)

    def weights(self):
        k = self.k
        codes = torch.stack((self.w & 15, self.w >> 4), 2).reshape(self.m, -1)[:, :k].double()
        wide = lambda t: t.double().repeat_interleave(self.group, 1)[:, :k]  # noqa: E731
        return (codes - (wide(self.z) if self.z is not None else 8.0)) * wide(self.s)

    def sums(self):
        """The products' sums, and the same of absolute values."""
        x = self.x[:, : self.k].double()
        if self.x8:
            x = x * self.x_scale.double()[:, None]
        w = self.weights()
        return x @ w.T, x.abs() @ w.abs().T

    def off(self):
        # A tensor core adds 16 exact products to a sum with at most 17 roundings of 2^-23 of the absolute values' sum; a group takes 8 such
        # steps at most, of three parts in fp32 24; then come K / 1024 + 1 groups' additions of 2^-24 a warp, four times as many of
        # groups of 32, 8 parts, and the scales' products.
        steps = 24 if self.dtype == K.THB_F32 and not self.x8 else 8
        return 17 * steps * 2.0 ** -23 + (4 * (self.k / 1024 + 1) + 12) * 2.0 ** -24


def check(layer, ref, slack):
    y, m, dtype = layer.y, layer.m, layer.dtype
    bound = slack + UNIT[dtype] * ref.abs() + 1e-30
    got = y[:, :m].double()
    assert bool(((got - ref).abs() <= bound).all()), float(((got - ref).abs() / bound).max())
    if dtype == K.THB_F32:  # (the bound above is the worst case; what is really lost is far less)
        assert float((got - ref).norm() / ref.norm()) < 2e-6
    pad = up(m, K.ALIGN[dtype])
    assert bool((y[:, m:pad] == 0).all()) and bool((y[:, pad:] == 7).all())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype,x8", [(K.THB_F32, False), (K.THB_F16, False), (K.THB_BF16, False), (K.THB_F16, True), (K.THB_F32, True)])
@pytest.mark.parametrize("m,k", [(1, 1), (16, 31), (17, 129), (40, 1000), (5, 8195), (333, 2048), (2400, 512), (4099, 640)])
def test_gemv_q4_sizes(lib, dtype, x8, group, m, k):
    for n in ((1, 8) if m * k > 100000 else (1, 2, 3, 5, 8)):
        layer = Layer(dtype, n, k, m, group, zeros=(n + k) % 2 == 0, x8=x8, sdtype=[K.THB_F16, K.THB_F32, K.THB_BF16][n % 3], seed=n)
        assert layer.call(lib) == 0
        torch.cuda.synchronize()
        ref, size = layer.sums()
        check(layer, ref, layer.off() * size)


@pytest.mark.parametrize("dtype", [K.THB_F32, K.THB_F16, K.THB_BF16])
@pytest.mark.parametrize("kind", [K.ACT_NONE, K.ACT_THRESHOLD, K.ACT_LEAKY, K.ACT_PRELU, K.ACT_SIGMOID, K.ACT_TANH])
def test_gemv_q4_epilogue(lib, dtype, kind):
    layer = Layer(dtype, 3, 300, 70, 64)
    layer.s *= 0.2
    scale, shift, slope = (torch.randn(70, device="cuda") for _ in range(3))
    d = layer.d
    d.scale, d.shift = scale.data_ptr(), shift.data_ptr()
    d.act.kind, d.act.threshold, d.act.value, d.act.alpha, d.act.slope = kind, 0.1, -0.5, 0.2, slope.data_ptr()
    assert layer.call(lib) == 0
    torch.cuda.synchronize()
    ref, size = layer.sums()
    v = ref * scale.double() + shift.double()
    slack = (layer.off() + 2.0 ** -23) * (size * scale.double().abs() + shift.double().abs())
    out = {K.ACT_NONE: v, K.ACT_THRESHOLD: torch.where(v > 0.1, v, -0.5), K.ACT_LEAKY: torch.where(v >= 0, v, 0.2 * v),
           K.ACT_PRELU: torch.where(v > 0, v, slope.double() * v), K.ACT_SIGMOID: torch.sigmoid(v), K.ACT_TANH: torch.tanh(v)}[kind]
    gain = torch.clamp(slope.double().abs(), min=1.0) if kind == K.ACT_PRELU else 1.0
    near = (v - 0.1).abs() <= slack if kind == K.ACT_THRESHOLD else torch.zeros_like(v, dtype=torch.bool)
    bound = slack * gain + UNIT[dtype] * out.abs() + 4e-7  # (expf and tanhf: 2 units in the last place of values up to 1, the division one)
    assert bool((((layer.y[:, :70].double() - out).abs() <= bound) | near).all())


def test_gemv_q4_range_of_fp32(lib):
    """fp32 rows of very large and very small values, infinities and NaN: a row's parts are its own."""
    layer = Layer(K.THB_F32, 6, 256, 48, 128, sdtype=K.THB_F32)
    layer.s.fill_(0.25)
    layer.x[1, :256] *= 1e34
    layer.x[2, :256] *= 1e-30
    layer.x[4, 7] = float("inf")
    layer.x[5, 200] = float("nan")
    assert layer.call(lib) == 0
    torch.cuda.synchronize()
    ref, size = layer.sums()
    got = layer.y[:, :48].double()
    assert bool(((got - ref)[:4].abs() <= (layer.off() * size + UNIT[K.THB_F32] * ref.abs())[:4]).all())
    for row in (4, 5):
        fine = torch.isfinite(ref[row])
        assert not bool(fine[:].all()) and torch.equal(torch.isnan(ref[row]), torch.isnan(got[row]))
        assert torch.equal(got[row][torch.isinf(ref[row])], ref[row][torch.isinf(ref[row])])


def test_gemv_q4_streams_and_graphs(lib):
    layer = Layer(K.THB_BF16, 4, 1024, 512, 32)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert layer.call(lib, s.cuda_stream) == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            assert layer.call(lib, s.cuda_stream) == 0
            assert layer.call(lib, s.cuda_stream) == 0
        layer.x[:, :1024] = torch.randn(4, 1024, device="cuda").to(torch.bfloat16)
        graph.replay()
    s.synchronize()
    ref, size = layer.sums()
    check(layer, ref, layer.off() * size)


def test_gemv_q4_of_quantized_weights(lib):
    """Weights through the host's quantiser and back through the product."""
    import numpy as np
    rng = np.random.default_rng(3)
    w = rng.standard_normal((50, 500)).astype(np.float32)
    layer = Layer(K.THB_F16, 8, 500, 50, 64, sdtype=K.THB_F32)
    codes, s, z = np.zeros((50, layer.d.w_ld), np.uint8), np.zeros((50, layer.d.s_ld), np.float32), np.zeros((50, layer.d.z_ld), np.uint8)
    assert lib.thb_q4_quantize_host(w.ctypes.data, 50, 500, 500, 64, 1, codes.ctypes.data, layer.d.w_ld, s.ctypes.data, layer.d.s_ld,
                                    z.ctypes.data, layer.d.z_ld) == 0
    layer.w.copy_(torch.from_numpy(codes)), layer.s.copy_(torch.from_numpy(s)), layer.z.copy_(torch.from_numpy(z))
    assert float((layer.weights().cpu() - torch.from_numpy(w).double()).abs().max()) <= 0.5 * float(s.max()) * 1.01
    assert layer.call(lib) == 0
    torch.cuda.synchronize()
    ref, size = layer.sums()
    check(layer, ref, layer.off() * size)


def test_gemv_q4_offsets_beyond_32_bits(lib):
    """More than 2^32 bytes of codes: the first, some middle and the last rows."""
    k, m, group = 32768, (1 << 32) // 16384 + 77, 128
    if torch.cuda.mem_get_info()[0] < 2 * m * k:
        pytest.skip("the device has no room for the weights")
    w = torch.zeros(m, k // 2, device="cuda", dtype=torch.uint8)
    some = torch.tensor([0, 31, 32, m // 2, m - 78, m - 33, m - 1], device="cuda")
    w[some] = torch.randint(0, 256, (7, k // 2), device="cuda", dtype=torch.uint8)
    s = torch.full((m, k // group), 0.01, device="cuda", dtype=torch.float16)
    x = torch.randn(2, k, device="cuda").half()
    y = torch.zeros(2, up(m, 8), device="cuda", dtype=torch.float16)
    d = K.GemvQ4Desc(dtype=K.THB_F16, N=2, K=k, M=m, group=group, x_ld=k, y_ld=y.stride(0), w_ld=k // 2, s_ld=k // group, wscale_dtype=K.THB_F16,
                     w=w.data_ptr(), wscale=s.data_ptr())
    assert lib.thb_gemv_q4_fwd(C.byref(d), x.data_ptr(), None, y.data_ptr(), None) == 0
    torch.cuda.synchronize()
    codes = torch.stack((w[some] & 15, w[some] >> 4), 2).reshape(7, k).double() - 8
    ws = codes * s[some].double().repeat_interleave(group, 1)
    ref, size = x.double() @ ws.T, x.double().abs() @ ws.abs().T
    bound = (17 * 8 * 2.0 ** -23 + (4 * (k / 1024 + 1) + 12) * 2.0 ** -24) * size + UNIT[K.THB_F16] * ref.abs()
    assert bool(((y[:, some].double() - ref).abs() <= bound).all())


def test_gemv_q4_of_weights_just_written(lib):
    """Codes, scales and zero points that the launch before in the stream writes, over and over: each product is of its own."""
    layer = Layer(K.THB_F16, 2, 4096, 2048, 64)
    g = torch.Generator(device="cuda").manual_seed(9)
    sets = [(torch.randint(0, 256, layer.w.shape, device="cuda", generator=g, dtype=torch.uint8), torch.rand(layer.s.shape, device="cuda", generator=g).half(),
             torch.randint(0, 16, layer.z.shape, device="cuda", generator=g, dtype=torch.uint8)) for _ in range(3)]
    got = []
    for i in range(60):
        layer.z.copy_(sets[i % 3][2]), layer.s.copy_(sets[i % 3][1]), torch.bitwise_or(sets[i % 3][0], 0, out=layer.w)
        assert layer.call(lib, torch.cuda.current_stream().cuda_stream) == 0
        got.append(layer.y.clone())
    torch.cuda.synchronize()
    for i in range(57):
        assert torch.equal(got[i], got[i + 3])
    for i in range(3):
        for t, src in zip((layer.w, layer.s, layer.z), sets[i]):
            t.copy_(src)
        layer.y.copy_(got[i])
        ref, size = layer.sums()
        check(layer, ref, layer.off() * size)
