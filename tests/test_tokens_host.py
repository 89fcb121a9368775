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
