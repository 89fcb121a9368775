"""Attention over values and keys that are not finite: a seen infinity or NaN shows in its own column of its own heads and nowhere else, scores of
-infinity weigh nothing, and what nobody sees is not looked at."""
import math

import pytest

torch = pytest.importorskip("torch")

from test_kv_append_gpu import EVERY
from test_paged_attn_gpu import Step
from thnets_b200 import kernels_abi as K

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lib():
    return K.load()


def put(step, row, position, head, d, k=None, v=None):
    page_len = step.cache.page_len
    page = int(step.cache.table[step.seq[row], position // page_len])
    for pool, rows, value in ((step.cache.k, step.k, k), (step.cache.v, step.v, v)):
        if value is not None:
            pool[page, position % page_len, head, d] = value
            rows[row][position, head, d] = value


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("lens", [[40, 200, 33], [3000, 1, 64]])
def test_attention_values_that_are_not_finite(lib, dtype, value, lens):
    step, plain = (Step(dtype, lens, 2, 6, 64, seed=3) for _ in range(2))
    put(step, 0, 17, 1, 5, v=value)
    assert step.call(lib) == 0 and plain.call(lib) == 0
    torch.cuda.synchronize()
    plain.check()
    got, ref = (s.y[:, : 6 * 64].float().reshape(3, 2, 3, 64).clone() for s in (step, plain))
    assert not bool(torch.isfinite(got[0, 1, :, 5]).any())
    got[0, 1, :, 5] = ref[0, 1, :, 5]
    assert torch.equal(got, ref) and torch.equal(step.lse, plain.lse)


@pytest.mark.parametrize("dtype", EVERY)
@pytest.mark.parametrize("lens", [[40, 200, 33], [3000, 1, 64]])
def test_attention_scores_of_minus_infinity(lib, dtype, lens):
    """A key of -infinity where q is positive: the token weighs nothing, as if it were not there."""
    step = Step(dtype, lens, 1, 2, 64, seed=4)
    step.q[0, [9, 64 + 9]] = 1.0
    for position in (0, 17, 39):
        put(step, 0, position, 0, 9, k=-math.inf)
    assert step.call(lib) == 0
    torch.cuda.synchronize()
    keep = [i for i in range(lens[0]) if i not in (0, 17, 39)]
    step.k[0], step.v[0] = step.k[0][keep], step.v[0][keep]
    step.check()


@pytest.mark.parametrize("dtype", EVERY)
def test_attention_without_a_score_above_minus_infinity(lib, dtype):
    step = Step(dtype, [3, 20], 1, 1, 64, seed=5)
    step.q[0, 9] = 1.0
    for position in range(3):
        put(step, 0, position, 0, 9, k=-math.inf)
    assert step.call(lib) == 0
    torch.cuda.synchronize()
    assert bool((step.y[0, :64] == 0).all()) and float(step.lse[0, 0]) == -math.inf
    step.lens[0], step.k[0], step.v[0] = 0, step.k[0][:0], step.v[0][:0]
    step.check()


@pytest.mark.parametrize("dtype", EVERY)
def test_attention_scores_of_infinity_and_nan(lib, dtype):
    """Their heads of the row are NaN, as the formula's; the others are not touched."""
    for value in (math.inf, math.nan):
        step, plain = (Step(dtype, [70, 50], 2, 4, 64, seed=6) for _ in range(2))
        for s in (step, plain):
            s.q[0, 9 : 256 : 64] = 1.0
        put(step, 0, 33, 0, 9, k=value)
        assert step.call(lib) == 0 and plain.call(lib) == 0
        torch.cuda.synchronize()
        assert bool(torch.isnan(step.y[0, :128]).all())
        assert torch.equal(step.y[0, 128:256], plain.y[0, 128:256]) and torch.equal(step.y[1], plain.y[1])
