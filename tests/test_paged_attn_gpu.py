"""Attention of one token over a paged cache against the formula in 64 bits: every type, shared and unshared heads, sizes of a head, both
orders and many sizes of a page, lengths from none to thousands, windows, rows of a padded batch, pages that do not exist.  Everything in the
pool that no row may see is NaN."""
import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

from test_kv_append_gpu import EVERY, TORCH, UNIT, Cache
from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return K.load()


class Step:
    def __init__(self, dtype, lens, heads, q_heads, dim, page_len=16, by_head=False, window=0, max_len=None, seq=None, scale=None, peak=1.0, seed=0):
        most = max(max(lens), 1)
        self.dtype, self.heads, self.q_heads, self.dim, self.window = dtype, heads, q_heads, dim, window
        self.lens, self.seq = lens, seq if seq is not None else list(range(len(lens)))
        seqs = max(self.seq) + 1
        self.cache = Cache(dtype, heads, dim, page_len, seqs, (most + page_len - 1) // page_len, by_head, seed=seed + 1)
        g = torch.Generator(device="cuda").manual_seed(seed)
        td = TORCH[dtype]
        self.cache.raw.fill_(float("nan"))
        self.k, self.v = [], []
        for row, n in enumerate(lens):
            n, start = max(n, 0), max(0, n - window) if window else 0
            k, v = (torch.randn(n, heads, dim, device="cuda", generator=g).to(td) for _ in range(2))
            at = torch.arange(start, n, device="cuda")
            pages = self.cache.table.long()[self.seq[row], at // page_len]
            self.cache.k[pages, at % page_len], self.cache.v[pages, at % page_len] = k[start:], v[start:]
            self.k.append(k[start:])
            self.v.append(v[start:])
        rows = len(lens)
        self.q = (peak * torch.randn(rows, q_heads * dim + 8, device="cuda", generator=g)).to(td)
        self.y = torch.full((rows, q_heads * dim + 16), 7.0, device="cuda", dtype=td)
        self.lse = torch.full((rows + 1, q_heads), 7.0, device="cuda")
        self.len_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.seq_t = torch.tensor(self.seq, dtype=torch.int32, device="cuda") if seq is not None else None
        self.scale = dim ** -0.5 if scale is None else scale
        d = self.d = K.PagedAttnDesc(cache=self.cache.desc, rows=rows, q_heads=q_heads, q_ld=self.q.stride(0), y_ld=self.y.stride(0), len=self.len_t.data_ptr(),
                                     seq=self.seq_t.data_ptr() if seq is not None else None, max_len=most if max_len is None else max_len, window=window,
                                     scale=self.scale, lse=self.lse.data_ptr())
        self.scratch = None

    def call(self, lib, stream=None):
        need = lib.thb_paged_attn_scratch(C.byref(self.d))
        if need and self.scratch is None:
            self.scratch = torch.full((need // 4,), float("nan"), device="cuda")  # (nothing in it has to be anything)
            self.d.scratch, self.d.scratch_bytes = self.scratch.data_ptr(), need
        return lib.thb_paged_attn_fwd(C.byref(self.d), self.q.data_ptr(), self.y.data_ptr(), stream)

    def check(self):
        worst = 0.0
        share, dim, dtype = self.q_heads // self.heads, self.dim, self.dtype
        for row, n in enumerate(self.lens):
            got = self.y[row, : self.q_heads * dim].double().reshape(self.heads, share, dim)
            lse = self.lse[row].double().reshape(self.heads, share)
            assert bool((self.y[row, self.q_heads * dim:] == 7).all())
            if n < 0:
                assert bool((got == 7).all()) and bool((lse == 7).all())
                continue
            if n == 0:
                assert bool((got == 0).all()) and bool((lse == -math.inf).all())
                continue
            q = self.q[row, : self.q_heads * dim].double().reshape(self.heads, share, dim)
            k, v = self.k[row].double().transpose(0, 1), self.v[row].double().transpose(0, 1)  # [heads][n][dim]
            s = self.scale * (q @ k.transpose(1, 2))
            p = torch.softmax(s, 2)
            y, size = p @ v, p @ v.abs()
            # A step of a tensor core on 16 products rounds its sum 17 times by 2^-23 of the absolute values' sum at most; a score takes
            # dim / 16 of them (fp32: six times as many), the scale and the base-2 exponent 2^-22 of it.  An error d of a score is a factor
            # 1 + d of its p.  p's parts hold 2^-16 of it, exp2 2^-22; a warp adds at most 34 tiles of twice (fp32: six times) 17
            # roundings, warps and chunks a few more; the division and the shrinking of the sums 2^-20 together.
            parts = 6 if dtype == K.THB_F32 else 1
            d = self.scale * (q.abs() @ k.abs().transpose(1, 2)) * 17 * parts * ((dim + 15) // 16) * 2.0 ** -23 + s.abs() * 2.0 ** -22
            d = d.amax(2, keepdim=True)
            off = size * (2 * d + (2.0 ** -16 if dtype != K.THB_F32 else 2.0 ** -22) + 17 * max(parts, 2) * 34 * 2.0 ** -23 + 2.0 ** -20)
            bound = off + UNIT[dtype] * y.abs() + (2.0 ** -25 if dtype == K.THB_F16 else 1e-37)
            assert bool(((got - y).abs() <= bound).all()), (row, n, float(((got - y).abs() / bound).max()))
            if dtype == K.THB_F32:  # (what is really lost is far less)
                assert float((got - y).norm() / size.norm()) < 1e-6
            ref = torch.logsumexp(s, 2)
            assert bool(((lse - ref).abs() <= 2 * d[:, :, 0] + 2.0 ** -21 * ref.abs() + 2.0 ** -15).all())
        assert bool((self.lse[len(self.lens)] == 7).all())


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("heads,q_heads,dim", [(1, 1, 64), (8, 32, 128), (12, 12, 80), (2, 20, 128), (1, 17, 64), (2, 4, 256), (3, 3, 8), (1, 8, 200), (4, 4, 136)])
def test_attention_heads(lib, dtype, heads, q_heads, dim):
    step = Step(dtype, [1, 700, 0, 130, -1, 33], heads, q_heads, dim)
    assert step.call(lib) == 0, lib.thb_last_cuda_error()
    torch.cuda.synchronize()
    step.check()
    assert int(step.cache.status) == 0


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("page_len", [1, 7, 16, 64, 1000])
@pytest.mark.parametrize("by_head", [False, True])
@pytest.mark.parametrize("window", [0, 1, 50, 5000])
def test_attention_pages_and_windows(lib, dtype, page_len, by_head, window):
    step = Step(dtype, [15, 16, 17, 63, 64, 65, 1, 129, 2100], 2, 6, 64, page_len, by_head, window)
    assert step.call(lib) == 0
    torch.cuda.synchronize()
    step.check()
    assert int(step.cache.status) == 0


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("rows,length,heads", [(1, 20000, 2), (1, 9001, 1), (40, 300, 4), (700, 40, 1), (3, 5000, 8)])
def test_attention_splits(lib, dtype, rows, length, heads):
    """One long row, many short ones, and lengths far below what max_len allows."""
    lens = [max(0, length - 37 * r) for r in range(rows)]
    step = Step(dtype, lens, heads, 4 * heads, 64, page_len=32, max_len=length + 100, peak=3.0)
    assert step.call(lib) == 0
    torch.cuda.synchronize()
    step.check()


@pytest.mark.parametrize("dtype", EVERY)
def test_attention_of_shared_sequences(lib, dtype):
    """Rows that name their sequences: two rows may read the same one."""
    step = Step(dtype, [400, 90, 0], 2, 2, 64, seq=[3, 0, 1])
    twice = Step(dtype, [400, 90, 0], 2, 2, 64, seq=[3, 0, 1])
    twice.seq_t[2], twice.len_t[2] = 3, 400
    twice.q[2] = twice.q[0]
    assert step.call(lib) == 0 and twice.call(lib) == 0
    torch.cuda.synchronize()
    step.check()
    assert torch.equal(twice.y[2], twice.y[0]) and torch.equal(twice.y[:2], step.y[:2]) and torch.equal(twice.lse[2], twice.lse[0])


@pytest.mark.parametrize("dtype", EVERY)
def test_attention_sharp_and_extreme_scores(lib, dtype):
    """One token takes all of the weight, or all take the same; scores far from zero on either side."""
    for peak, scale in ((30.0, 1.0), (1.0, 0.0), (40.0, -0.5)):
        step = Step(dtype, [1500, 64], 2, 4, 64, peak=peak, scale=scale)
        assert step.call(lib) == 0
        torch.cuda.synchronize()
        if abs(peak * scale) < 10:
            step.check()
        for row in range(2):
            q, k = step.q[row, :256].double().reshape(2, 2, 64), step.k[row].double().transpose(0, 1)
            p = torch.softmax(scale * (q @ k.transpose(1, 2)), 2)
            y = p @ step.v[row].double().transpose(0, 1)
            # check()'s bound with all 17 roundings of a step at their worst is useless for scores of some hundreds: two of them in effect
            steps = 4 * (6 if dtype == K.THB_F32 else 1)
            d = float((abs(scale) * (q.abs() @ k.abs().transpose(1, 2))).max()) * steps * 2 * 2.0 ** -23
            assert float((step.y[row, :256].double().reshape(2, 2, 64) - y).norm() / y.norm()) < 2 * UNIT[dtype] + 2.0 ** -16 + 2 * d


@pytest.mark.parametrize("dtype", EVERY)
def test_attention_small_weights_count(lib, dtype):
    """A first token of large weight and thousands of weight 2^-20 each, whose values are what the result consists of."""
    n, dim = 12000, 64
    step = Step(dtype, [n], 1, 1, dim, page_len=64, scale=math.log(2.0))
    k, v = step.k[0], step.v[0]
    k.zero_(), v.zero_()
    step.q.zero_()
    step.q[0, 0] = 1.0
    k[0, 0, 0] = 20.0
    v[1:, 0, 1] = 64.0
    at = torch.arange(n, device="cuda")
    pages = step.cache.table.long()[0, at // 64]
    step.cache.k[pages, at % 64], step.cache.v[pages, at % 64] = k, v
    assert step.call(lib) == 0
    torch.cuda.synchronize()
    ref = 64.0 * (n - 1) * 2.0 ** -20 / (1 + (n - 1) * 2.0 ** -20)
    assert abs(float(step.y[0, 1]) / ref - 1) < UNIT[dtype] + 2.0 ** -12 and float(step.y[0, 0]) == 0


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("bad", [-1, 10 ** 9, None])
def test_attention_bad_pages(lib, dtype, bad):
    """A page outside the pool is left out (its 16 positions do not count); None: the first page after the pool's last."""
    step = Step(dtype, [100, 100], 2, 2, 64)
    step.cache.table[0, 3] = step.cache.pages if bad is None else bad
    keep = [i for i in range(100) if i // 16 != 3]
    step.k[0], step.v[0] = step.k[0][keep], step.v[0][keep]
    assert step.call(lib) == 0
    torch.cuda.synchronize()
    step.check()
    assert int(step.cache.status) == -4


@pytest.mark.parametrize("dtype", EVERY)
def test_attention_bad_lengths_and_sequences(lib, dtype):
    step = Step(dtype, [96, 40, 80], 2, 2, 64, seq=[0, 1, 2])
    step.d.max_len = 80
    step.len_t[1] = 10 ** 9      # cut to max_len: sequence 1 has 40 positions of numbers, the rest of its pages are NaN
    step.seq_t[2] = 3            # no such sequence
    assert step.call(lib) == 0
    torch.cuda.synchronize()
    assert int(step.cache.status) == -4
    assert bool(torch.isnan(step.y[1, :128]).all()) and bool((step.y[2, :128] == 0).all()) and bool((step.lse[2] == -math.inf).all())
    step.lens[0], step.k[0], step.v[0] = 80, step.k[0][:80], step.v[0][:80]
    step.lens, step.k, step.v = step.lens[:1], step.k[:1], step.v[:1]
    step.lse[1] = 7
    step.check()


def test_attention_offsets_beyond_32_bits(lib):
    """A pool of more than 2^32 elements, its last pages in use."""
    heads, dim, page_len = 8, 128, 64
    pages = (1 << 32) // (heads * dim * page_len) + 3
    if torch.cuda.mem_get_info()[0] < 6 * pages * heads * dim * page_len:
        pytest.skip("the device has no room for the pool")
    k = torch.empty(pages, page_len, heads, dim, device="cuda", dtype=torch.float16)
    v = torch.empty_like(k)
    step = Step(K.THB_F16, [150], heads, heads, dim, page_len)
    step.cache.table.copy_(torch.tensor([[pages - 1, 0, pages - 2]]))
    at = torch.arange(150, device="cuda")
    where = step.cache.table.long()[0, at // 64]
    k[where, at % 64], v[where, at % 64] = step.k[0], step.v[0]
    c = step.d.cache
    c.pages, c.k, c.v, c.page_stride, c.token_stride, c.head_stride = pages, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2)
    assert step.call(lib) == 0
    torch.cuda.synchronize()
    step.check()


def test_attention_streams_and_graphs(lib):
    """Two calls with a scratch each on two streams, and a captured one replayed after the lengths have grown."""
    a, b = Step(K.THB_BF16, [3000, 10], 2, 8, 128), Step(K.THB_F16, [2500, 1, 700], 2, 2, 64, seed=5)
    for step in (a, b):
        assert step.call(lib) == 0
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    graphs = []
    for s, step in ((sa, a), (sb, b)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            assert step.call(lib, s.cuda_stream) == 0
        step.y.fill_(7), step.lse.fill_(7)
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(5):
        for s, g in ((sa, graphs[0]), (sb, graphs[1])):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    a.check(), b.check()
    a.len_t[0] = 1777
    a.lens[0], a.k[0], a.v[0] = 1777, a.k[0][:1777], a.v[0][:1777]
    graphs[0].replay()
    torch.cuda.synchronize()
    a.check()


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("dim", [64, 72, 96, 128, 160, 256])
@pytest.mark.parametrize("heads,q_heads,length,window", [(1, 16, 3000, 0), (2, 48, 900, 700), (8, 8, 5000, 0), (4, 28, 260, 0), (1, 1, 16500, 16400)])
def test_attention_one_row(lib, dtype, dim, heads, q_heads, length, window):
    """A single row, its length shared by as many CTAs as there may be: clusters of every size, a second launch, more than eight and more
    than sixteen heads a key head."""
    step = Step(dtype, [length], heads, q_heads, dim, page_len=32, window=window, seed=dim)
    assert step.call(lib) == 0, lib.thb_last_cuda_error()
    torch.cuda.synchronize()
    step.check()
    assert int(step.cache.status) == 0


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("max_len", [100, 4000, 40000])
def test_attention_rows_without_tokens(lib, dtype, max_len):
    """Only empty and padded rows, however the call is cut: zeros, and what was there."""
    step = Step(dtype, [0, -1, 0], 2, 4, 64, max_len=max_len, window=0)
    assert step.call(lib) == 0
    torch.cuda.synchronize()
    step.check()
