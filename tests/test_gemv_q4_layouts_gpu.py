"""4-bit Linear in the layouts and sizes that other tests leave out: scales and zero points with rows of just their groups, of multiples of four and
of eight and of odd lengths, at even and odd addresses; so many rows that a CTA has several tiles of 32, with reductions that one warp or several
share.  Against the formula in 64 bits."""
import pytest

torch = pytest.importorskip("torch")

from test_gemv_q4_gpu import Layer, check, up
from test_gemv_q4_order_gpu import repitch
from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.gpu

KINDS = [(K.THB_F32, False), (K.THB_F16, False), (K.THB_BF16, False), (K.THB_F16, True), (K.THB_BF16, True)]


@pytest.fixture(scope="module")
def lib():
    return K.load()


def product(lib, layer):
    assert layer.call(lib) == 0, lib.thb_last_cuda_error()
    torch.cuda.synchronize()
    ref, size = layer.sums()
    check(layer, ref, layer.off() * size)


@pytest.mark.parametrize("dtype,x8", KINDS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("sdtype", [K.THB_F16, K.THB_BF16, K.THB_F32])
def test_gemv_q4_pitches_of_scales(lib, dtype, x8, group, zeros, sdtype):
    for m, k in ((333, 2048), (100, 2050), (70, 9216), (5000, 1024), (40, 260)):
        groups = (k + group - 1) // group
        for s_ld, z_ld in ((groups, groups), (up(groups, 8), up(groups, 8)), (up(groups, 4), up(groups, 4) + 8), (groups | 1, groups + 1), (up(groups, 8), groups | 1)):
            product(lib, repitch(Layer(dtype, 3, k, m, group, zeros=zeros, x8=x8, sdtype=sdtype), s_ld, z_ld))


@pytest.mark.parametrize("sdtype", [K.THB_F16, K.THB_F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_gemv_q4_scales_anywhere(lib, group, sdtype, shift):
    """Scales that begin at a multiple of their own size only, zero points at any byte."""
    k, m = 2048, 300
    groups = k // group
    layer = repitch(Layer(K.THB_BF16, 2, k, m, group, sdtype=sdtype), groups, groups)
    s, z = torch.empty(m * groups + shift, device="cuda", dtype=layer.s.dtype), torch.empty(m * groups + shift, device="cuda", dtype=torch.uint8)
    s[shift:], z[shift:] = layer.s.flatten(), layer.z.flatten()
    layer.d.wscale, layer.d.wzero = s[shift:].data_ptr(), z[shift:].data_ptr()
    product(lib, layer)


@pytest.mark.parametrize("dtype,x8", KINDS)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,k", [(10007, 64), (10007, 1000), (32003, 96), (32003, 515), (9600, 2304), (14336, 1100)])
def test_gemv_q4_many_tiles_a_cta(lib, dtype, x8, group, zeros, m, k):
    groups = (k + group - 1) // group
    for n, s_ld in ((1, groups), (4, up(groups, 8)), (8, up(groups, 4))):
        product(lib, repitch(Layer(dtype, n, k, m, group, zeros=zeros, x8=x8, sdtype=K.THB_F16, seed=n), s_ld, s_ld))


@pytest.mark.parametrize("dtype", [K.THB_F32, K.THB_F16, K.THB_BF16])
@pytest.mark.parametrize("m,k", [(9999, 14400), (5100, 25100)])
def test_gemv_q4_many_tiles_with_x_from_memory(lib, dtype, m, k):
    """Rows of x that the shared memory has no room for, and several tiles a CTA."""
    for group in (32, 128):
        groups = (k + group - 1) // group
        product(lib, repitch(Layer(dtype, 8, k, m, group), groups, up(groups, 8)))
