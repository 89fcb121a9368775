"""A decoder of two layers, token by token, through the kernel ABI: norms with the residual, 4-bit projections, keys and values into the
paged cache, attention over it.  Against the same decoder in 64 bits from the same codes, run on all tokens at once; the second half of
the tokens through a captured graph of one step."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

from test_kv_append_gpu import TORCH, UNIT, Cache, rotated
from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.gpu

LAYERS, WIDTH, HEADS, Q_HEADS, DIM, HIDDEN, SEQS, STEPS, PAGE, EPS = 2, 256, 2, 8, 32, 640, 3, 40, 16, 1e-5


@pytest.fixture(scope="module")
def lib():
    return K.load()


def quantized(lib, w, group=32):
    """Codes, fp16 scales and zero points of fp32 weights on the device, and the weights that they stand for."""
    m, k = w.shape
    host = w.cpu().contiguous()
    codes = torch.zeros(m, (k + 31) // 32 * 16, dtype=torch.uint8)
    s, z = torch.zeros(m, k // group), torch.zeros(m, k // group, dtype=torch.uint8)
    assert lib.thb_q4_quantize_host(host.data_ptr(), m, k, k, group, 1, codes.data_ptr(), codes.shape[1], s.data_ptr(), s.shape[1], z.data_ptr(), z.shape[1]) == 0
    codes, s, z = codes.cuda(), s.half().cuda(), z.cuda()
    q = torch.stack((codes & 15, codes >> 4), 2).reshape(m, -1)[:, :k].double()
    return (codes, s, z), (q - z.double().repeat_interleave(group, 1)) * s.double().repeat_interleave(group, 1)


class Decoder:
    def __init__(self, lib, dtype, codes_between):
        self.lib, self.dtype, self.td, self.x8 = lib, dtype, TORCH[dtype], codes_between
        g = torch.Generator(device="cuda").manual_seed(11)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.freq = 10000.0 ** (-torch.arange(DIM // 2, dtype=torch.float64, device="cuda") / (DIM // 2))
        self.len = torch.zeros(SEQS, dtype=torch.int32, device="cuda")
        self.pos = torch.zeros(SEQS, dtype=torch.int32, device="cuda")
        shapes = dict(qkv=((Q_HEADS + 2 * HEADS) * DIM, WIDTH), out=(WIDTH, Q_HEADS * DIM), up=(HIDDEN, WIDTH), down=(WIDTH, HIDDEN))
        self.layers, self.keep = [], []
        for i in range(LAYERS):
            layer = dict(cache=Cache(dtype, HEADS, DIM, PAGE, SEQS, STEPS // PAGE + 1, seed=i), gains=[1 + 0.1 * rand(WIDTH) for _ in range(2)])
            for name, (m, k) in shapes.items():
                layer[name], layer[name + "_w"] = quantized(lib, rand(m, k) / math.sqrt(k))
            layer["slopes"] = (0.1 * rand(HIDDEN).abs()).contiguous()
            self.layers.append(layer)
        zeros = lambda n: torch.zeros(SEQS, n, device="cuda", dtype=self.td)  # noqa: E731
        self.x, self.stream_sum, self.delta = zeros(WIDTH), zeros(WIDTH), zeros(WIDTH)
        self.normed, self.qkv, self.q, self.att, self.hidden = zeros(WIDTH), zeros((Q_HEADS + 2 * HEADS) * DIM), zeros(Q_HEADS * DIM), zeros(Q_HEADS * DIM), zeros(HIDDEN)
        self.codes, self.scales = torch.zeros(SEQS, WIDTH, device="cuda", dtype=torch.float8_e4m3fn), torch.zeros(SEQS, device="cuda")

    def norm(self, x, res, gain, stream):
        d = K.RmsNormDesc(dtype=self.dtype, C=WIDTH, rows=SEQS, x_ld=WIDTH, res_ld=WIDTH, sum_ld=WIDTH, y_ld=WIDTH, q_ld=WIDTH, gain=gain.data_ptr(), eps=EPS)
        s = self.stream_sum
        assert self.lib.thb_rmsnorm_fwd(C.byref(d), x.data_ptr(), res.data_ptr() if res is not None else None, s.data_ptr(), None if self.x8 else self.normed.data_ptr(),
                                        self.codes.data_ptr() if self.x8 else None, self.scales.data_ptr() if self.x8 else None, stream) == 0

    def product(self, weights, x, y, stream, slopes=None, x8=False):
        codes, s, z = weights
        m, k = codes.shape[0], s.shape[1] * 32
        d = K.GemvQ4Desc(dtype=self.dtype, N=SEQS, K=k, M=m, group=32, x_ld=k, y_ld=m, w_ld=codes.shape[1], s_ld=s.shape[1], z_ld=z.shape[1],
                         wscale_dtype=K.THB_F16, w=codes.data_ptr(), wscale=s.data_ptr(), wzero=z.data_ptr())
        if slopes is not None:
            d.act.kind, d.act.slope = K.ACT_PRELU, slopes.data_ptr()
        assert self.lib.thb_gemv_q4_fwd(C.byref(d), (self.codes if x8 else x).data_ptr(), self.scales.data_ptr() if x8 else None, y.data_ptr(), stream) == 0

    def step(self, stream):
        """x of each sequence -> the residual stream after the last layer, in self.stream_sum."""
        res = None
        src = self.x
        size = self.x.element_size()
        for layer in self.layers:
            self.norm(src, res, layer["gains"][0], stream)
            self.product(layer["qkv"], self.normed, self.qkv, stream, x8=self.x8)
            at, ld = self.qkv.data_ptr(), self.qkv.stride(0)
            cache = layer["cache"].desc
            d = K.KvAppendDesc(cache=cache, rope=K.Rope(dim=DIM, freq=self.freq.data_ptr(), magnitude=1.0), tokens=SEQS, pos=self.pos.data_ptr(), k_ld=ld, v_ld=ld,
                               q_ld=ld, q_out_ld=Q_HEADS * DIM, q_heads=Q_HEADS)
            assert self.lib.thb_kv_append_fwd(C.byref(d), at + Q_HEADS * DIM * size, at + (Q_HEADS + HEADS) * DIM * size, at, self.q.data_ptr(), stream) == 0
            a = K.PagedAttnDesc(cache=cache, rows=SEQS, q_heads=Q_HEADS, q_ld=Q_HEADS * DIM, y_ld=Q_HEADS * DIM, len=self.len.data_ptr(), max_len=STEPS, scale=DIM ** -0.5)
            need = self.lib.thb_paged_attn_scratch(C.byref(a))
            if need and "scratch" not in layer:
                layer["scratch"] = torch.empty(need, dtype=torch.uint8, device="cuda")
            if need:
                a.scratch, a.scratch_bytes = layer["scratch"].data_ptr(), need
            assert self.lib.thb_paged_attn_fwd(C.byref(a), self.q.data_ptr(), self.att.data_ptr(), stream) == 0
            self.product(layer["out"], self.att, self.delta, stream)
            self.norm(self.delta, self.stream_sum, layer["gains"][1], stream)
            self.product(layer["up"], self.normed, self.hidden, stream, slopes=layer["slopes"], x8=self.x8)
            self.product(layer["down"], self.hidden, self.delta, stream)
            src, res = self.delta, self.stream_sum
        d = K.RmsNormDesc(dtype=self.dtype, C=WIDTH, rows=SEQS, x_ld=WIDTH, res_ld=WIDTH, sum_ld=WIDTH, eps=EPS)
        assert self.lib.thb_rmsnorm_fwd(C.byref(d), src.data_ptr(), res.data_ptr(), self.stream_sum.data_ptr(), None, None, None, stream) == 0

    def wide(self, x):
        """The same of all tokens at once, x [SEQS][STEPS][WIDTH], in 64 bits with nothing rounded on the way but codes of 8 bits."""
        def norm(t, gain):
            y = t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * gain.double()
            if not self.x8:
                return y
            s = y.abs().amax(-1, keepdim=True) / 448
            return (y / s).to(torch.float8_e4m3fn).double() * s

        pos = torch.arange(STEPS, device="cuda")
        mask = pos[None, :] > pos[:, None]
        for layer in self.layers:
            qkv = (norm(x, layer["gains"][0]) @ layer["qkv_w"].T).reshape(SEQS * STEPS, -1, DIM)
            turned, _ = rotated(qkv[:, : Q_HEADS + HEADS], pos.repeat(SEQS), self.freq, 1.0, DIM, False)
            split = lambda t, h: t.reshape(SEQS, STEPS, h, DIM).transpose(1, 2)  # noqa: E731
            q, k, v = split(turned[:, :Q_HEADS], Q_HEADS), split(turned[:, Q_HEADS:], HEADS), split(qkv[:, Q_HEADS + HEADS:], HEADS)
            k, v = (t.repeat_interleave(Q_HEADS // HEADS, 1) for t in (k, v))
            s = (q @ k.transpose(2, 3) * DIM ** -0.5).masked_fill(mask, -math.inf)
            x = x + (torch.softmax(s, 3) @ v).transpose(1, 2).reshape(SEQS, STEPS, -1) @ layer["out_w"].T
            h = norm(x, layer["gains"][1]) @ layer["up_w"].T
            x = x + torch.where(h > 0, h, layer["slopes"].double() * h) @ layer["down_w"].T
        return x


@pytest.mark.parametrize("codes_between", [False, True])
@pytest.mark.parametrize("dtype", [K.THB_F32, K.THB_F16, K.THB_BF16])
def test_decoder_token_by_token(lib, dtype, codes_between):
    dec = Decoder(lib, dtype, codes_between)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(SEQS, STEPS, WIDTH, device="cuda", generator=g).to(dec.td)
    got = []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for i in range(STEPS // 2):
            dec.x.copy_(x[:, i])
            dec.pos.fill_(i), dec.len.fill_(i + 1)
            dec.step(s.cuda_stream)
            got.append(dec.stream_sum.clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            dec.step(s.cuda_stream)
        for i in range(STEPS // 2, STEPS):
            dec.x.copy_(x[:, i])
            dec.pos.fill_(i), dec.len.fill_(i + 1)
            graph.replay()
            got.append(dec.stream_sum.clone())
    s.synchronize()
    assert all(int(layer["cache"].status) == 0 for layer in dec.layers)
    got, ref = torch.stack(got, 1).double(), dec.wide(x.double())
    # A layer rounds seven tensors on the way to the stream and the stream twice, each by a unit at most; a part's error passes through
    # the norm and the products with its relative size about kept, so that two layers are off by some 2 * 9 units in norm.  With codes
    # of 8 bits a value near a border may take the next code, 2^-3 of itself: an error e of its input does that to 8 e of the values, each off by
    # 2^-3, sqrt(8 e) * 2^-3 in norm a norm, four norms.
    e = 18 * UNIT[dtype]
    limit = e if not codes_between else e + 4 * math.sqrt(8 * e) / 8
    assert float((got - ref).norm() / ref.norm()) < limit


def first_calls_captured():
    """(in a process of its own)"""
    lib = K.load()
    for dtype, codes_between in ((K.THB_F16, True), (K.THB_F32, False)):
        captured, eager = Decoder(lib, dtype, codes_between), Decoder(lib, dtype, codes_between)
        for dec in (captured, eager):
            dec.x.copy_(torch.randn(SEQS, WIDTH, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)))
            dec.len.fill_(1)
        torch.cuda.synchronize()
        s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            captured.step(s.cuda_stream)
        graph.replay()
        eager.step(None)
        torch.cuda.synchronize()
        assert torch.equal(captured.stream_sum, eager.stream_sum) and bool((eager.stream_sum != 0).any())


def test_first_calls_of_a_process_captured():
    """Nothing that a first call sets up has to happen outside of a capture."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = "import sys; sys.path[:0] = [%r, %r]; import test_decoder_step_gpu as t; t.first_calls_captured()" % (here, os.path.dirname(here))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
