"""How precise attention over a context in two parts is in f32 for few rows, in the mean over a result (its tests elsewhere bound the worst element)."""
import numpy as np
import pytest

import floneum_amd as fa
from context_helpers import EPS, Call, definition

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [64, 80, 128, 192, 256])
@pytest.mark.parametrize("B, P, window, scale", [(2, 0, 1024, None), (2, 700, 0, None), (4, 700, 900, None), (2, 700, 0, 0.4)])
def test_few_f32_rows(device, D, B, P, window, scale):
    """The bound is on the root mean square.  Scores about nothing with a standard deviation of sigma = scale sqrt(D) are four sums of D / 4 products, each with D / 16
    roundings one after the other (the matrix instruction adds four products), then two that join them and one at the size of the distance from the largest: independent,
    of either sign, each 2^-24 / sqrt(3) of partial sums below sigma in the mean, so all of them together are below 2^-24 sigma sqrt(D / 16 + 3) / 2 with partial
    sums that grow to half of sigma.  The exponential, the sums of weights and the division add at most 4 steps of 2^-24.  A score's error reaches the weights as a relative
    one, and the result with the same size (values about nothing, so that weighted errors and weighted values add up alike)."""
    c = Call(device, fa.F32, B, 32, 8, 1, 1300, P, D, seed=D, scale=scale, lean=0.0)
    how = dict(offset=P + 1299, window=window, sinks=4)
    got = c.run(**how).astype(np.float64)
    want, _ = definition(c.q, c.k, c.v, c.pk, c.pv, c.scale, c.mask(**how), fa.F32, fa.F32)
    sigma = c.scale * np.sqrt(D)
    off = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert off <= EPS * (sigma * np.sqrt(D / 16 + 3) / 2 + 4)
