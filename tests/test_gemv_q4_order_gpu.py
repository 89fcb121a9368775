"""4-bit weights that the launch directly before the product writes: codes, scales and zero points, each in turn the last, by kernels that
rewrite them in place, in every layout of the scales (loads of one, of a block's and of eight groups)."""
import pytest

torch = pytest.importorskip("torch")

from test_gemv_q4_gpu import Layer, check
from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return K.load()


def repitch(layer, s_ld, z_ld):
    """Scales and zero points with rows of s_ld and z_ld entries."""
    groups = (layer.k + layer.group - 1) // layer.group
    for name, ld in (("s", s_ld), ("z", z_ld)):
        old = getattr(layer, name)
        if old is None:
            continue
        new = torch.full((layer.m, ld), 9, device="cuda").to(old.dtype)
        new[:, :groups] = old[:, :groups]
        setattr(layer, name, new)
    layer.d.wscale, layer.d.s_ld = layer.s.data_ptr(), s_ld
    if layer.z is not None:
        layer.d.wzero, layer.d.z_ld = layer.z.data_ptr(), z_ld
    return layer


@pytest.mark.parametrize("last", ["codes", "scales", "zeros"])
@pytest.mark.parametrize("group,pad", [(32, 0), (32, 4), (64, 1), (64, 2), (128, 0)])
@pytest.mark.parametrize("dtype,k,m", [(K.THB_F16, 4096, 2048), (K.THB_BF16, 12032, 512)])
def test_gemv_q4_of_what_the_launch_before_writes(lib, last, group, pad, dtype, k, m):
    groups = (k + group - 1) // group
    layer = repitch(Layer(dtype, 3, k, m, group), groups + pad, groups + pad)
    stream = torch.cuda.current_stream().cuda_stream
    flip = torch.randint(0, 256, layer.w.shape, device="cuda", dtype=torch.uint8)
    # (each is its own inverse, so that two states alternate; scales times -1: another sign of every product)
    write = {"codes": lambda: layer.w.bitwise_xor_(flip), "scales": lambda: layer.s.neg_(), "zeros": lambda: layer.z.bitwise_xor_(flip[:, : groups + pad])}
    got = []
    for _ in range(40):
        write[last]()
        assert layer.call(lib, stream) == 0
        got.append(layer.y.clone())
    torch.cuda.synchronize()
    for i in range(2):  # (the states of the last two calls are those of every second one)
        layer.y.copy_(got[39 - i])
        z = layer.z
        layer.z = z & 15  # (the low four bits count)
        ref, size = layer.sums()
        layer.z = z
        check(layer, ref, layer.off() * size)
        write[last]()
        for j in range(39 - i, -1, -2):
            assert torch.equal(got[j], got[39 - i])
    assert not torch.equal(got[0], got[1])
