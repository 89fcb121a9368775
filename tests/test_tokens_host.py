"""What the operators of a decoder's step refuse, and empty calls, without a GPU: every refusal comes before the first CUDA call."""
import ctypes as C
import os

import pytest

from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.skipif(not os.path.exists(K.DEFAULT_LIB), reason="libthnets.so not built")

AT = 1 << 20  # an address that is never followed
OK, UNSUPPORTED, ARG = 0, -1, -4


@pytest.fixture(scope="module")
def lib():
    return K.load()


def changed(make, **fields):
    d = make()
    for name, value in fields.items():
        setattr(d, name, value)
    return d


def norm_desc():
    return K.RmsNormDesc(dtype=K.THB_F16, C=100, rows=4, x_ld=104, res_ld=104, sum_ld=104, y_ld=104, q_ld=112, gain=AT, eps=1e-5)


def test_rmsnorm_refusals(lib):
    def call(d, x=AT, res=AT, total=AT, y=AT, q=AT, q_scale=AT):
        return lib.thb_rmsnorm_fwd(C.byref(d), x, res, total, y, q, q_scale, None)

    assert lib.thb_rmsnorm_fwd(None, AT, None, None, AT, None, None, None) == ARG
    for dtype in (K.THB_U8, 4, -1):
        assert call(changed(norm_desc, dtype=dtype)) == UNSUPPORTED
    assert call(changed(norm_desc, C=32769, x_ld=40000, res_ld=40000, sum_ld=40000, y_ld=40000, q_ld=40000)) == UNSUPPORTED
    assert b"32768" in lib.thb_last_cuda_error()
    for bad in (dict(rows=-1), dict(C=0), dict(eps=-1.0), dict(eps=float("nan")), dict(x_ld=96), dict(x_ld=108), dict(res_ld=0),
                dict(sum_ld=-104), dict(y_ld=99), dict(q_ld=104)):
        assert call(changed(norm_desc, **bad)) == ARG, bad
    for bad in (dict(x=None), dict(x=AT + 2), dict(res=AT + 8), dict(total=AT + 4), dict(y=AT + 8), dict(q=AT + 8), dict(q=None),
                dict(q_scale=None), dict(total=None, y=None, q=None, q_scale=None)):
        assert call(norm_desc(), **bad) == ARG, bad
    assert call(changed(norm_desc, rows=0)) == OK


def q4_desc():
    return K.GemvQ4Desc(dtype=K.THB_F16, N=2, K=100, M=30, group=32, x_ld=104, y_ld=32, w_ld=64, s_ld=4, z_ld=4, wscale_dtype=K.THB_F16,
                        w=AT, wscale=AT, wzero=AT)


def test_gemv_q4_refusals(lib):
    def call(d, x=AT, x_scale=None, y=AT):
        return lib.thb_gemv_q4_fwd(C.byref(d), x, x_scale, y, None)

    assert lib.thb_gemv_q4_fwd(None, AT, None, AT, None) == ARG
    for bad in (dict(dtype=K.THB_U8), dict(dtype=9), dict(N=9), dict(group=16), dict(group=0), dict(group=256), dict(wscale_dtype=K.THB_U8)):
        assert call(changed(q4_desc, **bad)) == UNSUPPORTED, bad
    for bad in (dict(N=-1), dict(K=0), dict(M=0), dict(x_ld=96), dict(x_ld=101), dict(y_ld=24), dict(y_ld=31), dict(w_ld=48), dict(w_ld=56),
                dict(s_ld=3), dict(z_ld=3), dict(w=None), dict(w=AT + 8), dict(wscale=None), dict(wscale=AT + 1),
                dict(act=K.Act(kind=6)), dict(act=K.Act(kind=-1)), dict(act=K.Act(kind=K.ACT_PRELU))):
        assert call(changed(q4_desc, **bad)) == ARG, bad
    for bad in (dict(x=None), dict(y=None), dict(x=AT + 8), dict(y=AT + 4), dict(x_scale=AT)):  # (with scales x_ld is a multiple of 16)
        assert call(q4_desc(), **bad) == ARG, bad
    assert call(changed(q4_desc, N=0)) == OK


@pytest.mark.parametrize("with_zero", [0, 1])
@pytest.mark.parametrize("k,group", [(1, 32), (100, 32), (257, 128), (64, 64)])
def test_q4_quantize_host(lib, with_zero, k, group):
    """The nearest code of every weight: half a step off at most, and the ends of a group are reached."""
    import numpy as np
    rng = np.random.default_rng(k)
    w = (rng.standard_normal((7, k + 3)) * np.exp(rng.standard_normal((7, 1)))).astype(np.float32)
    w[3, :k] = 0
    w[4, :k] = np.abs(w[4, :k])
    groups, ld = (k + group - 1) // group, (k + 1) // 2 + 5
    codes, s, z = np.full((7, ld), 255, np.uint8), np.full((7, groups + 1), 9, np.float32), np.full((7, groups + 2), 77, np.uint8)
    at = lambda a: a.ctypes.data  # noqa: E731
    assert lib.thb_q4_quantize_host(at(w), 7, k, k + 3, group, with_zero, at(codes), ld, at(s), groups + 1, at(z), groups + 2) == OK
    q = np.stack((codes & 15, codes >> 4), 2).reshape(7, -1)[:, :k].astype(np.float64)
    wide = lambda a: np.repeat(a[:, :groups], group, 1)[:, :k].astype(np.float64)  # noqa: E731
    zero = wide(z) if with_zero else 8.0
    got = (q - zero) * wide(s)
    # half a step, and where the zero point itself was rounded a range's end may be half a step beyond the last code
    assert np.all(np.abs(got - w[:, :k]) <= wide(s) * (1.0 if with_zero else 0.5) * (1 + 1e-6))
    assert np.all(s[:, groups] == 9) and np.all(z[:, groups:] == 77) and (with_zero or np.all(z == 77))
    assert np.all(got[3] == 0) and (with_zero or q.min() >= 1)
    w[0, 0] = np.inf
    assert lib.thb_q4_quantize_host(at(w), 7, k, k + 3, group, with_zero, at(codes), ld, at(s), groups + 1, at(z), groups + 2) == ARG
    for bad in ((None, 7, k, k + 3, group, 1, at(codes), ld, at(s), groups, at(z), groups), (at(w), 7, k, k - 1, group, 1, at(codes), ld, at(s), groups, at(z), groups),
                (at(w), 7, k, k, group, 1, at(codes), (k + 1) // 2 - 1, at(s), groups, at(z), groups), (at(w), 7, k, k, group, 1, at(codes), ld, at(s), groups, None, groups),
                (at(w), 7, k, k, group, 1, at(codes), ld, at(s), groups - 1, at(z), groups), (at(w), 7, k, k, 0, 1, at(codes), ld, at(s), groups, at(z), groups)):
        assert lib.thb_q4_quantize_host(*bad) == ARG


def cache_desc(**fields):
    c = K.KvCache(dtype=K.THB_F16, heads=4, dim=64, pages=10, page_len=16, page_stride=4096, token_stride=256, head_stride=64, k=AT, v=AT,
                  table=AT, table_ld=5, sequences=3, status=AT)
    for name, value in fields.items():
        setattr(c, name, value)
    return c


BAD_CACHES = (dict(heads=0), dict(dim=0), dict(dim=60), dict(dim=264), dict(dim=-64), dict(pages=0), dict(page_len=0), dict(table_ld=0),
              dict(sequences=0), dict(k=None), dict(v=None), dict(table=None), dict(status=None), dict(k=AT + 8), dict(v=AT + 2),
              dict(page_stride=4100), dict(token_stride=252), dict(head_stride=60), dict(page_stride=-4096), dict(token_stride=-256),
              dict(head_stride=-64), dict(token_stride=248), dict(head_stride=56), dict(page_stride=4088), dict(head_stride=128),
              dict(token_stride=64, head_stride=1016), dict(page_stride=1 << 41), dict(page_len=32))


def append_desc():
    return K.KvAppendDesc(cache=cache_desc(), rope=K.Rope(dim=64, freq=AT, magnitude=1.0), tokens=2, pos=AT, seq=AT, k_ld=256, v_ld=256,
                          q_ld=512, q_out_ld=512, q_heads=8)


def test_kv_append_refusals(lib):
    def call(d, k=AT, v=AT, q=AT, q_out=AT):
        return lib.thb_kv_append_fwd(C.byref(d), k, v, q, q_out, None)

    assert lib.thb_kv_append_fwd(None, AT, AT, AT, AT, None) == ARG
    for dtype in (K.THB_U8, 7):
        assert call(changed(append_desc, cache=cache_desc(dtype=dtype))) == UNSUPPORTED
    for bad in BAD_CACHES:
        assert call(changed(append_desc, cache=cache_desc(**bad))) == ARG, bad
    for bad in (dict(tokens=-1), dict(pos=None), dict(rope=K.Rope(dim=63, freq=AT)), dict(rope=K.Rope(dim=66, freq=AT)), dict(rope=K.Rope(dim=-2, freq=AT)),
                dict(rope=K.Rope(dim=64)), dict(q_heads=0), dict(q_ld=504), dict(q_out_ld=516), dict(k_ld=248), dict(v_ld=260), dict(seq=None, tokens=4)):
        assert call(changed(append_desc, **bad)) == ARG, bad
    for bad in (dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(k=AT + 8), dict(v=AT + 4), dict(q=AT + 2), dict(q_out=AT + 8),
                dict(k=None, v=None, q=None, q_out=None)):
        assert call(append_desc(), **bad) == ARG, bad
    assert call(changed(append_desc, cache=cache_desc(dim=60)), k=None, v=None) == ARG
    assert call(changed(append_desc, tokens=0)) == OK


def test_rope_freq_host(lib):
    import math

    import numpy as np
    out, mag = np.zeros(32), C.c_float()

    def call(dim=64, base=10000.0, scaling=K.ROPE_PLAIN, factor=4.0, trained=4096.0, slow=1.0, fast=32.0):
        out[:] = -1
        rc = lib.thb_rope_freq_host(dim, base, scaling, factor, trained, slow, fast, out.ctypes.data, C.byref(mag))
        return rc, out[: dim // 2].copy() if dim > 0 else None, mag.value

    plain = 10000.0 ** (-np.arange(32) / 32)
    assert call()[0] == OK and np.allclose(call()[1], plain, rtol=1e-14) and call()[2] == 1.0
    assert np.allclose(call(scaling=K.ROPE_LINEAR)[1], plain / 4, rtol=1e-14)
    # the raised base leaves the fastest pair and slows the last one by the whole factor
    raised = call(scaling=K.ROPE_BASE)[1]
    assert np.isclose(raised[0], plain[0]) and np.isclose(raised[31], plain[31] / 4) and np.all(np.diff(raised) < 0)
    rc, parts, m = call(scaling=K.ROPE_BY_PARTS)
    turns = 4096 * plain / (2 * math.pi)
    assert rc == OK and np.isclose(m, 0.1 * math.log(4) + 1)
    assert np.allclose(parts[turns >= 32], plain[turns >= 32]) and np.allclose(parts[turns <= 1], plain[turns <= 1] / 4)
    assert np.all(parts <= plain * (1 + 1e-12)) and np.all(parts >= plain / 4 * (1 - 1e-12)) and np.all(np.diff(parts) < 0)
    for bad in (dict(dim=0), dict(dim=63), dict(dim=-2), dict(base=0.0), dict(base=float("nan")), dict(scaling=1, factor=0.5), dict(scaling=2, factor=float("nan")),
                dict(scaling=3, trained=0.0), dict(scaling=3, slow=32.0), dict(scaling=3, slow=-1.0)):
        assert call(**bad)[0] == ARG, bad
    assert call(scaling=4)[0] == UNSUPPORTED and call(scaling=-1)[0] == UNSUPPORTED and call(dim=2, scaling=2)[0] == UNSUPPORTED
    assert call(dim=2)[0] == OK


def attn_desc():
    return K.PagedAttnDesc(cache=cache_desc(), rows=3, q_heads=8, q_ld=512, y_ld=520, len=AT, max_len=80, scale=0.1, scratch=AT, scratch_bytes=1 << 30)


def test_paged_attn_refusals(lib):
    def call(d, q=AT, y=AT):
        return lib.thb_paged_attn_fwd(C.byref(d), q, y, None)

    assert lib.thb_paged_attn_fwd(None, AT, AT, None) == ARG
    for dtype in (K.THB_U8, 7):
        assert call(changed(attn_desc, cache=cache_desc(dtype=dtype))) == UNSUPPORTED
    for bad in BAD_CACHES:
        assert call(changed(attn_desc, cache=cache_desc(**bad))) == ARG, bad
    for bad in (dict(rows=-1), dict(q_heads=0), dict(q_heads=6), dict(q_heads=-4), dict(q_ld=504), dict(q_ld=516), dict(y_ld=256), dict(y_ld=514), dict(len=None),
                dict(max_len=-1), dict(max_len=(1 << 30) + 1), dict(window=-1), dict(scale=float("inf")), dict(scale=float("nan")), dict(rows=4)):
        assert call(changed(attn_desc, **bad)) == ARG, bad
    for bad in (dict(q=None), dict(y=None), dict(q=AT + 8), dict(y=AT + 2)):
        assert call(attn_desc(), **bad) == ARG, bad
    assert call(changed(attn_desc, rows=0)) == OK
    # a long row is split among more CTAs than can join it by themselves: scratch is needed
    need = lib.thb_paged_attn_scratch(C.byref(changed(attn_desc, max_len=100000)))
    assert need > 0 and need % 4 == 0
    for bad in (dict(scratch=None), dict(scratch_bytes=need - 1), dict(scratch=AT + 8)):
        assert call(changed(attn_desc, max_len=100000, **bad)) == ARG, bad
    huge = cache_desc(heads=70000, token_stride=70000 * 64, page_stride=16 * 70000 * 64)
    assert call(changed(attn_desc, cache=huge, rows=100000, seq=AT, q_heads=70000, q_ld=70000 * 64, y_ld=70000 * 64)) == UNSUPPORTED


def test_paged_attn_scratch_covers_every_split(lib):
    """The size grows with the rows, is none where nothing is split, and holds what a call's CTAs write at most."""
    assert lib.thb_paged_attn_scratch(None) == 0
    for rows in (1, 3, 100, 5000):
        for max_len in (0, 1, 64, 65, 1000, 100000):
            for window in (0, 40):
                d = changed(attn_desc, rows=rows, max_len=max_len, window=window)
                need = lib.thb_paged_attn_scratch(C.byref(d))
                a_row = 8 * (64 + 2) * 4
                span = min(max_len, window or max_len)
                assert need % (rows * a_row) == 0 and need // (rows * a_row) <= max(1, (span + 63) // 64)
                assert need == 0 or need // (rows * a_row) > 1
