"""New tokens into a paged cache against the formula in 64 bits: both pairings, parts of a head that end inside a vector, both layouts of
the pool, pages of one token to many, positions up to 10^9, padded places, pages and sequences that do not exist.  The whole pool is
compared: what no token owns stays as it was."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.gpu

UNIT = {K.THB_F32: 2.0 ** -24, K.THB_F16: 2.0 ** -11, K.THB_BF16: 2.0 ** -8}
TORCH = {K.THB_F32: torch.float32, K.THB_F16: torch.float16, K.THB_BF16: torch.bfloat16}
EVERY = [K.THB_F32, K.THB_F16, K.THB_BF16]


@pytest.fixture(scope="module")
def lib():
    return K.load()


class Cache:
    """A pool of pages in one of both orders, with gaps between pages, full of sevens; tables of pages in no order."""

    def __init__(self, dtype, heads, dim, page_len, seqs, a_seq, by_head=False, pool=None, seed=1):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype, self.heads, self.dim, self.page_len, self.by_head = dtype, heads, dim, page_len, by_head
        self.pages = pool or seqs * a_seq + 2
        gap = 8
        self.raw = torch.full((2, self.pages, heads * page_len * dim + gap), 7.0, device="cuda", dtype=TORCH[dtype])
        self.table = torch.randperm(self.pages, device="cuda", generator=g)[: seqs * a_seq].reshape(seqs, a_seq).to(torch.int32).contiguous() if pool is None \
            else (torch.arange(seqs * a_seq, device="cuda") % pool).reshape(seqs, a_seq).to(torch.int32)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        shape = (heads, page_len, dim) if by_head else (page_len, heads, dim)
        view = self.raw[..., : heads * page_len * dim].unflatten(2, shape)
        self.k, self.v = (t.transpose(1, 2) if by_head else t for t in view)  # [pages][page_len][heads][dim] either way
        self.desc = K.KvCache(dtype=dtype, heads=heads, dim=dim, pages=self.pages, page_len=page_len, page_stride=self.k.stride(0),
                              token_stride=self.k.stride(1), head_stride=self.k.stride(2), k=self.k.data_ptr(), v=self.v.data_ptr(),
                              table=self.table.data_ptr(), table_ld=a_seq, sequences=seqs, status=self.status.data_ptr())


def rotated(x, pos, freq, magnitude, rot, interleaved):
    """x: [tokens, heads, dim] in 64 bits."""
    angle = (pos.double()[:, None] * freq[: rot // 2])[:, None, :]
    cos, sin = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude
    out = x.clone()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, a * sin + b * cos
    size = x.abs()
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * magnitude
    return out, size


def near(got, ref, size, dtype):
    # cos and sin are off by 2^-23 from rounding and a last place or two of the function, the angle's fraction of a turn by 2^-24 of
    # half a turn, fp64 angles of 10^9 by 2^-21.5: 2^-20.5 of the pair's size; two products and a sum add 2^-22
    bound = 2.0 ** -20 * size + UNIT[dtype] * ref.abs() + 2.0 ** -25
    assert bool(((got.double() - ref).abs() <= bound).all()), float(((got.double() - ref).abs() / bound).max())


def run(lib, dtype, heads, q_heads, dim, page_len, seqs, a_seq, pos, seq, rot, interleaved, by_head=False, magnitude=1.0, base=10000.0, stream=None, pool=None):
    cache = Cache(dtype, heads, dim, page_len, seqs, a_seq, by_head, pool)
    tokens, td = len(pos), TORCH[dtype]
    g = torch.Generator(device="cuda").manual_seed(tokens + dim)
    width = (q_heads + 2 * heads) * dim
    qkv = torch.randn(tokens, width + 8, device="cuda", generator=g).to(td)
    pos_t = torch.tensor(pos, dtype=torch.int32, device="cuda")
    seq_t = torch.tensor(seq, dtype=torch.int32, device="cuda") if seq is not None else None
    freq = base ** (-2.0 * torch.arange(max(rot // 2, 1), dtype=torch.float64, device="cuda") / max(rot, 1))
    q_out = torch.full((tokens, q_heads * dim + 8), 7.0, device="cuda", dtype=td)
    size = qkv.element_size()
    d = K.KvAppendDesc(cache=cache.desc, rope=K.Rope(dim=rot, interleaved=int(interleaved), freq=freq.data_ptr() if rot else None, magnitude=magnitude),
                       tokens=tokens, pos=pos_t.data_ptr(), seq=seq_t.data_ptr() if seq is not None else None, k_ld=width + 8, v_ld=width + 8,
                       q_ld=width + 8, q_out_ld=q_heads * dim + 8, q_heads=q_heads)
    at = qkv.data_ptr()
    before = [cache.k.clone(), cache.v.clone()]
    rc = lib.thb_kv_append_fwd(C.byref(d), at + q_heads * dim * size, at + (q_heads + heads) * dim * size, at, q_out.data_ptr(), stream)
    torch.cuda.synchronize()
    assert rc == 0, lib.thb_last_cuda_error()
    rows = qkv[:, :width].double().reshape(tokens, -1, dim)
    turned, scale = rotated(rows[:, : q_heads + heads], pos_t, freq, magnitude, rot, interleaved)
    live = pos_t >= 0
    seqv = seq_t.long() if seq is not None else torch.arange(tokens, device="cuda")
    slot = pos_t.long() // page_len
    there = live & (seqv >= 0) & (seqv < seqs) & (slot < a_seq)
    page = cache.table.long()[seqv.clamp(0, seqs - 1), slot.clamp(0, a_seq - 1)]
    there &= (page >= 0) & (page < cache.pages)
    near(q_out[live, : q_heads * dim], turned[live, :q_heads].flatten(1), scale[live, :q_heads].flatten(1), dtype)
    assert bool((q_out[~live] == 7).all()) and bool((q_out[:, q_heads * dim:] == 7).all())
    inside = pos_t.long() % page_len
    near(cache.k[page[there], inside[there]], turned[there, q_heads:], scale[there, q_heads:], dtype)
    assert torch.equal(cache.v[page[there], inside[there]], qkv[:, :width].reshape(tokens, -1, dim)[there, q_heads + heads:])
    for got, was in ((cache.k, before[0]), (cache.v, before[1])):
        was[page[there], inside[there]] = got[page[there], inside[there]]
        assert torch.equal(got, was)
    assert bool((cache.raw[:, :, heads * page_len * dim:] == 7).all())
    assert int(cache.status) == (0 if bool((there == live).all()) else -4)
    return cache, qkv, q_out


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,q_heads,dim,rot", [(1, 1, 8, 8), (2, 6, 64, 64), (3, 3, 80, 40), (8, 32, 128, 128), (1, 5, 96, 6), (2, 2, 128, 24),
                                                   (4, 4, 256, 256), (2, 4, 64, 0), (1, 2, 40, 2), (1, 2, 256, 0), (2, 3, 256, 64), (2, 2, 80, 20), (1, 40, 256, 6),
                                                   (20, 20, 32, 32)])
def test_append_heads_and_rotations(lib, dtype, interleaved, heads, q_heads, dim, rot):
    run(lib, dtype, heads, q_heads, dim, 16, 3, 4, pos=[0, 17, 63], seq=None, rot=rot, interleaved=interleaved, by_head=rot % 3 == 0)


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("page_len", [1, 5, 16, 100])
@pytest.mark.parametrize("by_head", [False, True])
def test_append_prompts(lib, dtype, page_len, by_head):
    """Three prompts of different lengths in one call, beginning inside a page."""
    pos, seq = [], []
    for b, (start, n) in enumerate(((0, 1), (3, 130), (41, 57))):
        pos += list(range(start, start + n))
        seq += [b] * n
    run(lib, dtype, 2, 4, 64, page_len, 3, 133 // page_len + 1, pos, seq, 32, False, by_head, magnitude=1.25)


@pytest.mark.parametrize("dtype", EVERY)
def test_append_padded_and_bad_places(lib, dtype):
    """Places in a padded batch; sequences and positions beyond the table."""
    cache, _, _ = run(lib, dtype, 2, 2, 64, 16, 2, 3, pos=[-1, 5, -7, 47], seq=[0, 1, 99, 0], rot=64, interleaved=False)
    assert int(cache.status) == 0
    for pos, seq in (([5, 48], [0, 0]), ([5, 6], [0, 2]), ([5, 6], [-1, 0]), ([2 ** 31 - 1, 6], [0, 0])):
        cache, _, _ = run(lib, dtype, 2, 2, 64, 16, 2, 3, pos=pos, seq=seq, rot=64, interleaved=False)
        assert int(cache.status) == -4


@pytest.mark.parametrize("bad", [-1, 10 ** 9, 8])
def test_append_bad_pages(lib, bad, monkeypatch):
    """A table that names a page outside the pool (which has 8): the token is not written, its queries are rotated all the same."""
    made = Cache.__init__

    def spoilt(self, *a, **kw):
        made(self, *a, **kw)
        self.table[1, 2] = bad

    monkeypatch.setattr(Cache, "__init__", spoilt)
    cache, _, _ = run(lib, K.THB_F16, 2, 2, 64, 16, 2, 3, pos=[40, 40, 10], seq=[0, 1, 1], rot=64, interleaved=False)
    assert int(cache.status) == -4


@pytest.mark.parametrize("dtype", [K.THB_F32, K.THB_BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_far_positions(lib, dtype, interleaved):
    run(lib, dtype, 1, 2, 64, 128, 1, 10 ** 9 // 128 + 1, pos=[999_999_999, 1_000_003, 131_072], seq=[0, 0, 0], rot=64, interleaved=interleaved, pool=3)


def test_append_offsets_beyond_32_bits(lib):
    """A pool of more than 2^32 elements: a page near its end."""
    heads, dim, page_len = 8, 128, 64
    need = 2 * ((1 << 32) // (heads * dim * page_len) + 3) * heads * dim * page_len * 2
    if torch.cuda.mem_get_info()[0] < 3 * need:
        pytest.skip("the device has no room for the pool")
    pages = need // 4 // (heads * dim * page_len)
    k = torch.zeros(pages, page_len, heads, dim, device="cuda", dtype=torch.float16)
    v = torch.zeros_like(k)
    assert k.numel() > 1 << 32
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device="cuda")
    status, pos = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([63], dtype=torch.int32, device="cuda")
    kv = torch.randn(2, 1, heads * dim, device="cuda").half()
    c = K.KvCache(dtype=K.THB_F16, heads=heads, dim=dim, pages=pages, page_len=page_len, page_stride=k.stride(0), token_stride=k.stride(1),
                  head_stride=k.stride(2), k=k.data_ptr(), v=v.data_ptr(), table=table.data_ptr(), table_ld=1, sequences=1, status=status.data_ptr())
    d = K.KvAppendDesc(cache=c, rope=K.Rope(dim=0), tokens=1, pos=pos.data_ptr(), k_ld=heads * dim, v_ld=heads * dim)
    assert lib.thb_kv_append_fwd(C.byref(d), kv[0].data_ptr(), kv[1].data_ptr(), None, None, None) == 0
    torch.cuda.synchronize()
    assert torch.equal(k[-1, 63].flatten(), kv[0, 0]) and torch.equal(v[-1, 63].flatten(), kv[1, 0])
    assert int(torch.count_nonzero(k[-1, :63])) == 0 and int(torch.count_nonzero(k[0])) == 0 and int(status) == 0


def test_append_queries_alone_in_place_and_captured(lib):
    """Rotation without a cache, in place, in a captured graph on another stream."""
    x = torch.randn(5, 4 * 64, device="cuda").half()
    was = x.clone()
    freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device="cuda") / 32)
    pos = torch.tensor([0, 3, -1, 9, 1000], dtype=torch.int32, device="cuda")
    d = K.KvAppendDesc(cache=K.KvCache(dtype=K.THB_F16, dim=64), rope=K.Rope(dim=64, freq=freq.data_ptr(), magnitude=1.0), tokens=5, pos=pos.data_ptr(),
                       q_ld=256, q_out_ld=256, q_heads=4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            assert lib.thb_kv_append_fwd(C.byref(d), None, None, x.data_ptr(), x.data_ptr(), s.cuda_stream) == 0
        pos.copy_(torch.tensor([1, 3, -1, 9, 1000], dtype=torch.int32))
        graph.replay()
    s.synchronize()
    ref, size = rotated(was.double().reshape(5, 4, 64), pos, freq, 1.0, 64, False)
    ref[2] = was[2].double().reshape(4, 64)
    near(x.reshape(5, 4, 64), ref, size, K.THB_F16)
