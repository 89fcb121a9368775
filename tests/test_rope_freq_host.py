"""Frequencies scaled by parts, between the turns that keep them and those that divide them: in proportion to the turns, pair by pair."""
import ctypes as C
import math
import os

import numpy as np
import pytest

from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.skipif(not os.path.exists(K.DEFAULT_LIB), reason="libthnets.so not built")


@pytest.mark.parametrize("dim,base,factor,trained,slow,fast", [(64, 10000.0, 4.0, 4096.0, 1.0, 32.0), (128, 500000.0, 8.0, 8192.0, 1.0, 4.0), (128, 10000.0, 16.0, 2048.0, 0.0, 64.0),
                                                               (2, 10000.0, 2.0, 8.0, 1.0, 2.0)])
def test_rope_freq_by_parts_between_its_ends(dim, base, factor, trained, slow, fast):
    out, magnitude = np.zeros(dim // 2), C.c_float()
    assert K.load().thb_rope_freq_host(dim, base, K.ROPE_BY_PARTS, factor, trained, slow, fast, out.ctypes.data, C.byref(magnitude)) == 0
    between = 0
    for i in range(dim // 2):
        plain = base ** (-2.0 * i / dim)
        turns = trained * plain / (2 * math.pi)
        keep = min(max((turns - slow) / (fast - slow), 0.0), 1.0)
        assert math.isclose(out[i], plain * (keep + (1 - keep) / factor), rel_tol=1e-13)
        between += 0 < keep < 1
    assert between >= 1 and math.isclose(magnitude.value, 0.1 * math.log(factor) + 1, rel_tol=2.0 ** -23)
