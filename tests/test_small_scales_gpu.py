"""flash_attention at scales down to f32's smallest numbers: the weights of all visible keys are alike."""
import numpy as np
import pytest

import floneum_amd as fa
from q8_helpers import HALF_STEP, rounded, upload

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [fa.F32, fa.F16, fa.BF16])
@pytest.mark.parametrize("D", [64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("Sq", [1, 5, 150, 700])
@pytest.mark.parametrize("scale", [1e-44, 1e-39, 1e-37, 1e-20])
def test_weights_are_alike(device, dtype, D, Sq, scale):
    rng = np.random.default_rng(D + Sq)
    B, H, Hkv, Skv = 1, 4, 2, 800
    q, k, v = (rounded(rng.standard_normal(s).astype(np.float32), dtype) for s in ((B, H, Sq, D), (B, Hkv, Skv, D), (B, Hkv, Skv, D)))
    got = upload(device, q, dtype).flash_attention(*(upload(device, x, dtype) for x in (k, v)), scale, analytic=(True, Skv - Sq, 0)).to_numpy()
    seen = np.arange(Skv)[None] <= Skv - Sq + np.arange(Sq)[:, None]
    weights = seen / seen.sum(-1, keepdims=True)
    values = v.astype(np.float64).repeat(H // Hkv, 1)
    want, mass = weights @ values, weights @ np.abs(values)
    # half a step of the result; weights within half a step of the tensors' type; sums of n weights and of n products in f32, and the division
    bound = HALF_STEP[dtype] * np.abs(want) + (HALF_STEP[dtype] + 2.0 ** -24 * (2 * Skv / 16 + 16)) * mass
    assert (np.abs(np.asarray(got, np.float64) - want) <= bound).all()
