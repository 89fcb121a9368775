"""Results in the place of inputs: allowed row by row, refused where the rows of the two lie apart differently, before the first CUDA call."""
import ctypes as C
import os

import pytest

from test_tokens_host import ARG, AT, append_desc, changed, norm_desc, q4_desc
from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.skipif(not os.path.exists(K.DEFAULT_LIB), reason="libthnets.so not built")
FAR = [AT + (i << 20) for i in range(1, 8)]


@pytest.fixture(scope="module")
def lib():
    return K.load()


@pytest.mark.parametrize("place", ["total", "y"])
@pytest.mark.parametrize("of", ["x", "res"])
def test_rmsnorm_in_place_of_another_pitch(lib, place, of):
    at = dict(x=FAR[0], res=FAR[1], total=FAR[2], y=FAR[3], q=FAR[4], q_scale=FAR[5])
    at[place] = at[of]
    d = changed(norm_desc, **{("sum_ld" if place == "total" else "y_ld"): 112})
    assert lib.thb_rmsnorm_fwd(C.byref(d), *at.values(), None) == ARG
    assert b"place" in lib.thb_last_cuda_error()


def test_rmsnorm_results_in_one_place(lib):
    for at in ((FAR[0], FAR[1], FAR[2], FAR[2], None, None), (FAR[0], FAR[1], FAR[2], FAR[3], FAR[2], FAR[5]), (FAR[0], FAR[1], None, FAR[3], FAR[3], FAR[5]),
               (FAR[0], FAR[1], None, None, FAR[0], FAR[5]), (FAR[0], FAR[1], None, None, FAR[1], FAR[5])):
        assert lib.thb_rmsnorm_fwd(C.byref(norm_desc()), *at, None) == ARG, at
        assert b"place" in lib.thb_last_cuda_error()


def test_kv_append_in_place_of_another_pitch(lib):
    d = changed(append_desc, q_out_ld=520)
    assert lib.thb_kv_append_fwd(C.byref(d), FAR[0], FAR[1], FAR[2], FAR[2], None) == ARG
    assert b"place" in lib.thb_last_cuda_error()


def test_gemv_q4_in_place(lib):
    d = changed(q4_desc, y_ld=104)
    assert lib.thb_gemv_q4_fwd(C.byref(d), FAR[0], None, FAR[0], None) == ARG
    assert b"place" in lib.thb_last_cuda_error()
