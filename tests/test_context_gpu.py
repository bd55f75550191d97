"""Attention over a context in two parts on a GPU, against its definition in 64 bits."""
import numpy as np
import pytest

import floneum_amd as fa
from context_helpers import Call, spread, upload

pytestmark = pytest.mark.gpu
TYPES = [fa.F32, fa.F16, fa.BF16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 64, 72, 96, 128, 160, 256])
@pytest.mark.parametrize("B, H, Hkv, Sq, Skv, window, sinks", [(1, 4, 2, 1, 300, 100, 4), (2, 4, 1, 3, 333, 64, 70), (1, 2, 2, 40, 517, 129, 5)])
def test_sinks(device, dtype, D, B, H, Hkv, Sq, Skv, window, sinks):
    Call(device, dtype, B, H, Hkv, Sq, Skv, 0, D, seed=D).both(offset=Skv - Sq, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("B, H, Hkv, Sq, Skv, P", [(3, 4, 2, 1, 40, 300), (5, 6, 1, 2, 70, 129), (2, 2, 2, 33, 50, 200), (9, 8, 2, 1, 17, 513)])
def test_prefix(device, dtype, D, B, H, Hkv, Sq, Skv, P):
    rng = np.random.default_rng(P)
    lens = rng.integers(Sq, Skv + 1, B)
    Call(device, dtype, B, H, Hkv, Sq, Skv, P, D, seed=D).both(lens=lens, positions=lens - Sq, offset=P)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 4, 50])
@pytest.mark.parametrize("window, sinks", [(100, 4), (300, 260), (20, 1), (1, 0), (5, 5)])
def test_prefix_window_sinks(device, dtype, Sq, window, sinks):
    lens = np.asarray([60, 200, Sq])
    Call(device, dtype, 3, 4, 2, Sq, 200, 250, 128, seed=Sq).both(lens=lens, positions=lens - Sq, offset=250, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 3, 40])
def test_rows_without_a_key(device, dtype, Sq):
    """Lengths of nothing and below, positions in front of all keys, lengths beyond the cache."""
    c = Call(device, dtype, 5, 4, 2, Sq, 90, 0, 64, seed=3)
    c.both(lens=[0, -5, 90, 1000, 1], positions=[0, 0, -200, 5, 0], offset=50, window=30, sinks=2)
    c.both(lens=[0, -5, 90, 1000, 1], positions=[0, 0, -200, 5, 0], offset=50)
    c = Call(device, dtype, 3, 4, 2, Sq, 90, 33, 64, seed=3)
    c.both(lens=[0, -5, 90], positions=[-1000, 0, 30], offset=20, window=7, sinks=1)


@pytest.mark.parametrize("dtype", TYPES)
def test_no_own_keys_and_no_keys(device, dtype):
    c = Call(device, dtype, 2, 4, 2, 1, 0, 77, 64)
    c.both(causal=False)
    q, none = upload(device, np.ones((1, 2, 3, 64)), dtype), fa.Tensor.empty(device, (1, 2, 0, 64), dtype)
    got = q.flash_attention(none, none, 1.0, sinks=1, analytic=(True, 0, 4)).to_numpy()
    assert not got.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 40])
def test_without_a_causal_mask(device, dtype, Sq):
    Call(device, dtype, 2, 4, 2, Sq, 90, 130, 128).both(causal=False)
    Call(device, dtype, 2, 4, 2, Sq, 90, 130, 128).both(causal=False, offset=150, window=20, sinks=9)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 5, 64])
@pytest.mark.parametrize("D", [64, 33])
def test_layouts(device, dtype, Sq, D):
    """Heads behind rows in memory, gaps between rows, dims that do not lie side by side, and results likewise."""
    c = Call(device, dtype, 2, 4, 2, Sq, 150, 70, D, seed=1)
    how = dict(offset=70 + 150 - Sq, window=90, sinks=3)
    values = [c.q, c.k, c.v, c.pk[None], c.pv[None]]
    first = c.run(**how)
    c.check(first, **how)
    for order in ([0, 2, 1, 3], [3, 0, 1, 2], [1, 2, 0, 3]):
        got = c.run(tensors=[upload(device, x, dtype, order) for x in values], **how)
        c.check(got, **how)
    for steps in ([1, 1, 2, 1], [1, 2, 1, 1], [1, 1, 1, 2]):
        whole, out = spread(device, c.shape, dtype, steps, 7.0)
        c.check(c.run(out=out, **how), **how)
        left = np.ones(whole.shape, bool)
        left[tuple(slice(None, None, s) for s in steps)] = False
        rest = whole.to_numpy()[left]
        assert np.unique(rest).size <= 1  # nothing is written beside the result


@pytest.mark.parametrize("dtype", [fa.F16, fa.BF16])
@pytest.mark.parametrize("Sq", [1, 40])
def test_f32_results(device, dtype, Sq):
    Call(device, dtype, 2, 4, 2, Sq, 150, 70, 128).both(out_dtype=fa.F32, offset=220 - Sq, window=90, sinks=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 3.0])
@pytest.mark.parametrize("Sq", [1, 40])
def test_scales(device, dtype, scale, Sq):
    Call(device, dtype, 2, 4, 2, Sq, 150, 70, 64, scale=scale).both(offset=220 - Sq, window=90, sinks=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 40])
def test_same_tensor_twice(device, dtype, Sq):
    """Keys that are the values too, and a prefix that is the cache of one sequence."""
    c = Call(device, dtype, 1, 4, 2, Sq, 100, 100, 64, seed=9)
    c.v, c.pk, c.pv = c.k, c.k[0], c.k[0]
    k = upload(device, c.k, dtype)
    how = dict(offset=200 - Sq)
    c.check(c.run(tensors=[upload(device, c.q, dtype), k, k, k, k], **how), **how)
