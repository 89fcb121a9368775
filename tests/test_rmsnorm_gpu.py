"""Root-mean-square norm against the formula in 64 bits: every type, rows of a vector to rows of 32768 values, ends inside a vector,
pitches beyond the row, results in place, rows of zeros, of infinities and of NaN."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.gpu

UNIT = {K.THB_F32: 2.0 ** -24, K.THB_F16: 2.0 ** -11, K.THB_BF16: 2.0 ** -8}
TINY = {K.THB_F32: 2.0 ** -150, K.THB_F16: 2.0 ** -25, K.THB_BF16: 2.0 ** -134}  # half the least subnormal
TORCH = {K.THB_F32: torch.float32, K.THB_F16: torch.float16, K.THB_BF16: torch.bfloat16}
EVERY = [K.THB_F32, K.THB_F16, K.THB_BF16]


@pytest.fixture(scope="module")
def lib():
    return K.load()


def up(v, m):
    return (v + m - 1) // m * m


def call(lib, dtype, c, x, res=None, total=None, y=None, q=None, q_scale=None, gain=None, eps=1e-5, stream=None):
    d = K.RmsNormDesc(dtype=dtype, C=c, rows=x.shape[0], x_ld=x.stride(0), eps=eps)
    for name, t in (("res_ld", res), ("sum_ld", total), ("y_ld", y), ("q_ld", q)):
        setattr(d, name, t.stride(0) if t is not None else 0)
    d.gain = gain.data_ptr() if gain is not None else None
    at = [t.data_ptr() if t is not None else None for t in (x, res, total, y, q, q_scale)]
    return lib.thb_rmsnorm_fwd(C.byref(d), *at, stream)


def formula(x, res, gain, eps):
    t = x.double() + (res.double() if res is not None else 0)
    v = t / torch.sqrt((t * t).mean(1, keepdim=True) + eps)
    return t, v * gain.double() if gain is not None else v


def check(dtype, c, t, v, total, y, q, q_scale):
    # the sum's terms are positive: a thread adds 128 squares at most, warps and blocks ten times more, each rounding of 2^-24 of
    # the sum at most, half of that in the root; the root itself, the mean, the addition of eps and two products take eight more
    off = (128 + 10) / 2 * 2.0 ** -24 + 8 * 2.0 ** -24
    if total is not None:
        assert bool(((total[:, :c].double() - t).abs() <= (UNIT[dtype] + 2.0 ** -24) * t.abs() + TINY[dtype]).all())
    if y is not None:
        assert bool(((y[:, :c].double() - v).abs() <= (UNIT[dtype] * (1 + off) + off) * v.abs() + TINY[dtype]).all())
    if q is not None:
        top = v.abs().amax(1)
        assert bool(((q_scale.double() - top / 448).abs() <= (off + 2.0 ** -23) * top / 448).all())
        got = q[:, :c].double() * q_scale.double()[:, None]
        step = torch.maximum(2.0 ** -4 * v.abs(), 2.0 ** -10 * q_scale.double()[:, None])
        assert bool(((got - v).abs() <= step * (1 + 2.0 ** -12) + off * v.abs()).all())


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 7), (700, 16), (129, 64), (5, 130), (1, 264), (77, 1004), (3, 4096), (1300, 4096),
                                    (9, 5001), (4, 8200), (2, 16384), (3, 20001), (2, 32768)])
def test_rmsnorm_sizes(lib, dtype, rows, c):
    td, al = TORCH[dtype], K.ALIGN[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows * 40000 + c)
    ld = up(c, al) + 2 * al
    x = torch.randn(rows, ld, device="cuda", generator=g).to(td)
    res = (3 * torch.randn(rows, ld, device="cuda", generator=g)).to(td)
    x[:, c:], res[:, c:] = float("nan"), float("inf")  # what lies behind a row is not read into it
    gain = torch.randn(c, device="cuda", generator=g)
    total = torch.full((rows, ld), 7.0, device="cuda", dtype=td)
    y = torch.full((rows, ld + al), 7.0, device="cuda", dtype=td)
    q = torch.full((rows, up(c, 16) + 16), 7.0, device="cuda").to(torch.float8_e4m3fn)
    q_scale = torch.full((rows + 1,), 7.0, device="cuda")
    assert call(lib, dtype, c, x, res, total, y, q, q_scale, gain) == 0
    torch.cuda.synchronize()
    t, v = formula(x[:, :c], res[:, :c], gain, 1e-5)
    check(dtype, c, t, v, total, y, q, q_scale[:rows])
    for out, pad in ((total, up(c, al)), (y, up(c, al)), (q.float(), up(c, 16))):
        assert bool((out[:, c:pad].float() == 0).all()) and bool((out[:, pad:].float() == 7).all())
    assert float(q_scale[rows]) == 7.0
    # each result by itself is the same, and so are those that replace their inputs
    y1, q1, s1 = torch.full_like(y, 7.0), torch.full((rows, up(c, 16) + 16), 7.0, device="cuda").to(q.dtype), torch.empty_like(q_scale)
    assert call(lib, dtype, c, x, res, y=y1, gain=gain) == 0
    assert call(lib, dtype, c, x, res, q=q1, q_scale=s1, gain=gain) == 0
    res1, x1 = res.clone(), x.clone()
    assert call(lib, dtype, c, x1, res1, total=res1, y=x1, gain=gain) == 0
    torch.cuda.synchronize()
    assert torch.equal(y1, y) and torch.equal(q1.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s1[:rows], q_scale[:rows])
    assert torch.equal(res1[:, :c], total[:, :c]) and torch.equal(x1[:, :c], y[:, :c])


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("c", [40, 3000])
def test_rmsnorm_special_rows(lib, dtype, c):
    """Rows of zeros, an infinity, a NaN, values near the type's ends; the rows beside them are as without them."""
    td, al = TORCH[dtype], K.ALIGN[dtype]
    big = {K.THB_F32: 1e17, K.THB_F16: 6e4, K.THB_BF16: 1e17}[dtype]
    small = {K.THB_F32: 1e-35, K.THB_F16: 1e-7, K.THB_BF16: 1e-35}[dtype]
    g = torch.Generator(device="cuda").manual_seed(c)
    x = torch.randn(9, up(c, al), device="cuda", generator=g).to(td)
    x[:, c:] = 0
    x[1] = 0
    x[3, 5] = float("inf")
    x[5, c - 1] = float("nan")
    x[7] = big * torch.sign(x[7])
    x[8] = small * torch.sign(x[8])
    y, q, s = torch.empty_like(x), torch.empty(9, up(c, 16), device="cuda", dtype=torch.float8_e4m3fn), torch.empty(9, device="cuda")
    assert call(lib, dtype, c, x, y=y, q=q, q_scale=s, eps=1e-6) == 0
    torch.cuda.synchronize()
    fine = [0, 2, 4, 6, 7, 8]
    t, v = formula(x[fine, :c], None, None, 1e-6)
    check(dtype, c, t, v, None, y[fine], None, None)
    keep = [i for i in range(6) if not (dtype != K.THB_F16 and fine[i] == 8)]
    check(dtype, c, t[keep], v[keep], None, None, q[fine][keep], s[fine][keep])
    assert float(s[1]) == 0 and bool((q[1].float() == 0).all()) and bool((y[1] == 0).all())
    if dtype != K.THB_F16:  # 1e-35 / sqrt(1e-6) is below 2^-100
        assert float(s[8]) == 0 and bool((q[8].float() == 0).all())
    assert bool(torch.isnan(s[[3, 5]]).all())
    assert bool(torch.isnan(y[5, :c]).all()) and bool(torch.isnan(y[3, 5])) and bool((y[3, :5] == 0).all())


def test_rmsnorm_empty_and_streams(lib):
    """No rows; a stream of the caller's; a captured call replayed on other values."""
    x = torch.randn(6, 512, device="cuda").half()
    y = torch.zeros_like(x)
    d = K.RmsNormDesc(dtype=K.THB_F16, C=512, rows=0, x_ld=512, y_ld=512, eps=1e-5)
    assert lib.thb_rmsnorm_fwd(C.byref(d), x.data_ptr(), None, None, y.data_ptr(), None, None, None) == 0
    torch.cuda.synchronize()
    assert bool((y == 0).all())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert call(lib, K.THB_F16, 512, x, y=y, stream=s.cuda_stream) == 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            assert call(lib, K.THB_F16, 512, x, y=y, stream=s.cuda_stream) == 0
        x.copy_(torch.randn(6, 512, device="cuda"))
        graph.replay()
    s.synchronize()
    t, v = formula(x, None, None, 1e-5)
    check(K.THB_F16, 512, t, v, None, y, None, None)


def test_rmsnorm_offsets_beyond_32_bits(lib):
    """More than 2^32 values: the first and the last rows."""
    rows, c = (1 << 32) // 4096 + 5, 4096
    if torch.cuda.mem_get_info()[0] < 6 * rows * c:
        pytest.skip("the device has no room for the rows")
    x = torch.zeros(rows, c, device="cuda", dtype=torch.float16)
    ends = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    x[ends] = torch.randn(5, c, device="cuda").half()
    y = torch.full_like(x, 7.0)
    assert call(lib, K.THB_F16, c, x, y=y) == 0
    torch.cuda.synchronize()
    t, v = formula(x[ends], None, None, 1e-5)
    check(K.THB_F16, c, t, v, None, y[ends], None, None)
    assert bool((y[2:1000] == 0).all()) and bool((y[rows - 1000:rows - 2] == 0).all())
