"""Prompts into a paged cache: so many tokens that a warp has all heads of one (2368 and more on 148 SMs), in several trips of the heads that it
has under way, whose number divides the heads or does not; and few tokens of many heads, which several warps share.  The whole pool is
compared with the formula in 64 bits."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from test_kv_append_gpu import EVERY, TORCH, near, rotated, run
from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return K.load()


def prompts(tokens, seqs):
    """Positions and sequences of `seqs` prompts side by side, which begin at different places of a page."""
    return [t // seqs + 3 * (t % seqs) for t in range(tokens)], [t % seqs for t in range(tokens)]


# heads, q_heads, dim, rotated: units of 16 bytes and whole halves, parts of a head, halves of 8, 4 and 2 bytes, nothing turned
SHAPES = [(8, 32, 128, 128), (8, 25, 128, 64), (12, 12, 80, 80), (12, 12, 80, 40), (12, 13, 80, 20), (5, 12, 80, 10), (4, 50, 64, 64), (3, 17, 96, 6), (4, 7, 256, 192),
          (8, 32, 128, 0), (1, 90, 40, 40), (40, 40, 32, 32)]


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,q_heads,dim,rot", SHAPES)
def test_append_warp_to_a_token(lib, dtype, interleaved, heads, q_heads, dim, rot):
    pos, seq = prompts(2411, 3)
    pos[700] = pos[2410] = -1
    run(lib, dtype, heads, q_heads, dim, 64, 3, 13, pos, seq, rot, interleaved, by_head=dim == 80, magnitude=1.125)


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens", [1, 70, 600, 1300])
@pytest.mark.parametrize("heads,q_heads,dim,rot", [(16, 128, 128, 128), (24, 72, 64, 32), (20, 41, 80, 10)])
def test_append_warps_share_a_token(lib, dtype, interleaved, tokens, heads, q_heads, dim, rot):
    pos, seq = prompts(tokens, 2)
    run(lib, dtype, heads, q_heads, dim, 32, 2, 23, pos, seq, rot, interleaved)


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("q_heads,dim,rot", [(49, 128, 128), (49, 80, 40), (60, 80, 10)])
def test_append_queries_of_prompts_in_place(lib, dtype, interleaved, q_heads, dim, rot):
    tokens = 2400
    g = torch.Generator(device="cuda").manual_seed(dim + rot)
    x = torch.randn(tokens, q_heads * dim + 8, device="cuda", generator=g).to(TORCH[dtype])
    was = x.clone()
    freq = 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device="cuda") / rot)
    pos = torch.randint(0, 100000, (tokens,), device="cuda", generator=g, dtype=torch.int32)
    d = K.KvAppendDesc(cache=K.KvCache(dtype=dtype, dim=dim), rope=K.Rope(dim=rot, interleaved=int(interleaved), freq=freq.data_ptr(), magnitude=1.0), tokens=tokens,
                       pos=pos.data_ptr(), q_ld=x.stride(0), q_out_ld=x.stride(0), q_heads=q_heads)
    assert lib.thb_kv_append_fwd(C.byref(d), None, None, x.data_ptr(), x.data_ptr(), None) == 0
    torch.cuda.synchronize()
    ref, size = rotated(was[:, : q_heads * dim].double().reshape(tokens, q_heads, dim), pos, freq, 1.0, rot, interleaved)
    near(x[:, : q_heads * dim].reshape(tokens, q_heads, dim), ref, size, dtype)
    assert torch.equal(x[:, q_heads * dim:], was[:, q_heads * dim:])
