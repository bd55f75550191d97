"""Attention over a context in two parts: elements that are not finite, and scales, at every width of its kernels.  Against the definition in 64 bits
(context_helpers)."""
import numpy as np
import pytest

import floneum_amd as fa
from context_helpers import Call, definition, rounded

pytestmark = pytest.mark.gpu
TYPES = [fa.F32, fa.F16, fa.BF16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq, Skv, P", [(1, 300, 0), (1, 40, 200), (3, 90, 130), (140, 200, 130)])
@pytest.mark.parametrize("window, sinks", [(0, 0), (30, 5), (60, 37)])
@pytest.mark.parametrize("D", [8, 40, 56, 72, 80, 88, 104, 120, 136, 160, 184, 200, 248])
def test_infinite_keys_at_padded_head_dims(device, dtype, D, window, sinks, Sq, Skv, P):
    """A key whose score is -inf has no weight, also where the kernel's rows are wider than head_dim and where the first tokens end inside a tile."""
    c = Call(device, dtype, 2, 4, 2, Sq, Skv, P, D, seed=D)
    c.q[..., 0] = np.abs(c.q[..., 0]) + rounded(np.float32(0.25), dtype)
    how = dict(offset=P + Skv - Sq, window=window, sinks=sinks)
    for keys, at in ((c.pk[None] if P else c.k, 3), (c.k, Skv - 2)):
        keys[:, :, at, 0] = -np.inf
    got = c.run(**how)
    for keys, at in ((c.pk[None] if P else c.k, 3), (c.k, Skv - 2)):
        keys[:, :, at, 0] = 0.0
    seen = c.mask(**how)
    seen[:, :, [3, P + Skv - 2]] = False
    want, bound = definition(c.q, c.k, c.v, c.pk, c.pv, c.scale, seen, dtype, dtype)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 72, 96, 128, 192, 256])
@pytest.mark.parametrize("scale", [1e-44, 1e-39, 1e-30, 1e-15, 1e-4, 1.5, 40.0])
@pytest.mark.parametrize("Sq", [2, 150])
def test_any_scale(device, dtype, D, scale, Sq):
    """Scales down to f32's smallest numbers (the weights are then all alike) and such as leave one key all of the weight."""
    Call(device, dtype, 1, 4, 2, Sq, 200, 70, D, scale=scale, seed=D).both(offset=270 - Sq, window=190, sinks=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 136])
@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
@pytest.mark.parametrize("Sq", [2, 150])
def test_scales_at_the_end_of_f32(device, dtype, D, scale, Sq):
    """Scales whose product with log2 e is beyond f32, on queries and keys small enough for it (in f16, which has no such elements, on queries of nothing)."""
    c = Call(device, dtype, 1, 4, 2, Sq, 200, 70, D, scale=scale, std=3e-19 if dtype != fa.F16 else 1.0, lean=0.0, seed=D)
    if dtype == fa.F16:
        c.q[:] = 0.0
    c.both(offset=270 - Sq, window=190, sinks=3)
