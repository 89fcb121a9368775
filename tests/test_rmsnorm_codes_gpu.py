"""The norm's e4m3 codes against the formula in 64 bits, code by code: v / q_scale rounded to fp32 and that to e4m3, however near it is to
the border of two codes.  Rows made of borders, few and so many that a block has several, rows of ordinary values, rows too small for
448 / max|t * gain| in fp32."""
import pytest

torch = pytest.importorskip("torch")

from test_rmsnorm_gpu import EVERY, TORCH, call, up
from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return K.load()


def borders():
    """The 126 positive values half way between neighbouring codes (the largest code is 448)."""
    codes = torch.arange(127, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
    return (codes[1:] + codes[:-1]) / 2


def formula(x, res, gain):
    """What the codes stand for before a row's scale: t * gain / max|t * gain| * 448 (the root is common to a row)."""
    t = x.double() + (res.double() if res is not None else 0)
    w = t * gain.double() if gain is not None else t
    most = w.abs().amax(1, keepdim=True)
    return (w * (448.0 / most)).float().to(torch.float8_e4m3fn), w, most[:, 0]


def same(got, ref):
    """Equal as values: zero has two codes."""
    a, b = got.float(), ref.float()
    bad = (a != b) & ~(torch.isnan(a) & torch.isnan(b))
    assert not bool(bad.any()), (int(bad.sum()), a[bad][:5].tolist(), b[bad][:5].tolist())


def outputs(rows, c, dtype):
    q = torch.full((rows, up(c, 16) + 16), 7.0, device="cuda").to(torch.float8_e4m3fn)
    return q, torch.full((rows + 1,), 7.0, device="cuda")


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("with_gain", [False, True])
@pytest.mark.parametrize("rows,c", [(513, 16), (300, 63), (129, 255), (300, 1004), (200, 4096), (40, 9000), (5, 20001), (3, 32768),
                                    (40001, 16), (20003, 255), (7001, 1004), (2501, 2500), (2003, 4096), (1001, 9000), (603, 20001), (401, 32768)])
def test_codes_at_borders(lib, dtype, with_res, with_gain, rows, c):
    """Every value is a border of two codes, or beside one by a unit of fp32, by the gain or by what the residual adds."""
    td, al = TORCH[dtype], K.ALIGN[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows * 100003 + c)
    pick = lambda a, *s: a[torch.randint(0, a.numel(), s, device="cuda", generator=g)]  # noqa: E731
    ld = up(c, al) + al
    # fp16 holds 2^-10 to 448 as they are; the other types have rows of many sizes
    spread = pick(torch.tensor([1.0] if dtype == K.THB_F16 else [1.0, 2.0 ** 40, 2.0 ** -50, 2.0 ** -12], device="cuda", dtype=torch.float64), rows, 1)
    want = pick(borders(), rows, c) * torch.sign(torch.randn(rows, c, device="cuda", generator=g, dtype=torch.float64))
    want[:, c // 2] = 448.0
    if dtype == K.THB_F32:
        want *= 1 + pick(torch.tensor([0.0, 2.0 ** -23, -2.0 ** -23, 2.0 ** -22], device="cuda", dtype=torch.float64), rows, c)
        spread = spread * torch.exp(torch.rand(rows, 1, device="cuda", generator=g, dtype=torch.float64))  # (448 / max is no power of two)
    x = torch.full((rows, ld), float("nan"), device="cuda", dtype=td)
    x[:, :c] = (want * spread).to(td)
    res = None
    if with_res:  # less than fp32 holds beside x, or nothing
        res = torch.full((rows, ld), float("nan"), device="cuda", dtype=td)
        part = pick(torch.tensor([0.0, 2.0 ** -23, -2.0 ** -24, 2.0 ** -26, -2.0 ** -30], device="cuda", dtype=torch.float64), rows, c)
        res[:, :c] = (x[:, :c].double() * part).to(td)
    gain = pick(torch.tensor([1.0, 1 + 2.0 ** -23, 1 - 2.0 ** -24, 1 + 2.0 ** -22], device="cuda"), c).contiguous() if with_gain else None
    ref, _, _ = formula(x[:, :c], res[:, :c] if with_res else None, gain)
    for eps in (1e-5, 1e-12):
        q, s = outputs(rows, c, dtype)
        assert call(lib, dtype, c, x, res, q=q, q_scale=s, gain=gain, eps=eps) == 0
        torch.cuda.synchronize()
        same(q[:, :c], ref)
        assert bool((q[:, c:up(c, 16)].float() == 0).all()) and bool((q[:, up(c, 16):].float() == 7).all()) and float(s[rows]) == 7
    # with the other results, which replace their inputs
    x1, res1 = x.clone(), res.clone() if with_res else None
    q, s1 = outputs(rows, c, dtype)
    assert call(lib, dtype, c, x1, res1, total=res1, y=x1, q=q, q_scale=s1, gain=gain, eps=1e-12) == 0
    y, total = torch.empty_like(x), torch.empty_like(x)
    assert call(lib, dtype, c, x, res, total=total if with_res else None, y=y, gain=gain, eps=1e-12) == 0
    torch.cuda.synchronize()
    same(q[:, :c], ref)
    assert torch.equal(s1, s) and torch.equal(x1[:, :c], y[:, :c]) and (not with_res or torch.equal(res1[:, :c], total[:, :c]))


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("rows,c", [(30000, 128), (777, 1004), (3000, 4096), (500, 16384)])
def test_codes_of_ordinary_rows(lib, dtype, with_res, rows, c):
    td = TORCH[dtype]
    g = torch.Generator(device="cuda").manual_seed(c)
    x = (0.3 * torch.randn(rows, up(c, 8), device="cuda", generator=g)).to(td)
    res = (torch.randn(rows, up(c, 8), device="cuda", generator=g) * torch.exp(0.8 * torch.randn(up(c, 8), device="cuda", generator=g))).to(td) if with_res else None
    gain = (1 + 0.2 * torch.randn(c, device="cuda", generator=g)).contiguous()
    q, s = outputs(rows, c, dtype)
    assert call(lib, dtype, c, x, res, q=q, q_scale=s, gain=gain) == 0
    torch.cuda.synchronize()
    same(q[:, :c], formula(x[:, :c], res[:, :c] if with_res else None, gain)[0])


@pytest.mark.parametrize("dtype", [K.THB_F32, K.THB_BF16])
@pytest.mark.parametrize("small", ["values", "gain", "both"])
@pytest.mark.parametrize("c", [40, 1000, 5000])
def test_codes_of_tiny_rows(lib, dtype, small, c):
    """max|t * gain| where fp32 has no 448 / max, with a small eps that makes ordinary values of v: codes and scales of the formula, zeros zeros."""
    td, al = TORCH[dtype], K.ALIGN[dtype]
    g = torch.Generator(device="cuda").manual_seed(c)
    x = torch.randn(6, up(c, al), device="cuda", generator=g)
    x[:, 3::7] = 0
    x[:, c:] = 0
    gain = torch.randn(c, device="cuda", generator=g).contiguous()
    size, scale, eps = {"values": (1e-37, 1.0, 1e-20), "gain": (1e-10, 1e-27, 1e-20), "both": (1e-14, 1e-26, 1e-25)}[small]
    x, gain = (x * size).to(td), gain * scale
    q, s = outputs(6, c, dtype)
    y = torch.empty(6, up(c, al), device="cuda", dtype=td)
    assert call(lib, dtype, c, x, y=y, q=q, q_scale=s, gain=gain, eps=eps) == 0
    torch.cuda.synchronize()
    ref, w, most = formula(x[:, :c], None, gain)
    root = torch.sqrt((x[:, :c].double() ** 2).mean(1) + eps)
    top = most / root
    # fp32 sums of squares that are below 2^-126 are lost beside eps: at most 2^-126 / eps of the sum under the root
    off = (128 + 10) / 2 * 2.0 ** -24 + 12 * 2.0 ** -24 + 2.0 ** -126 / eps
    for row in range(6):
        if float(top[row]) >= 2.0 ** -100 * (1 + off):
            same(q[row:row + 1, :c], ref[row:row + 1])
            assert abs(float(s[row]) * 448 / float(top[row]) - 1) <= off
        elif float(top[row]) < 2.0 ** -100 * (1 - off):
            assert float(s[row]) == 0 and bool((q[row, :c].float() == 0).all())
    assert bool((q[:, 3:c:7].float() == 0).all()) and bool((q[:, c:up(c, 16)].float() == 0).all())
