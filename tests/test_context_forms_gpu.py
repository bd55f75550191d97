"""Attention over a context in two parts on every launch that its plan chooses: the calls of context_forms, whose forms are asserted, against the definition in 64
bits (context_helpers)."""
import numpy as np
import pytest

import floneum_amd as fa
from context_forms import CALLS_16, CALLS_F32, described
from context_helpers import Call
from test_context_forms import call

pytestmark = pytest.mark.gpu


def check(device, dtype, shape, form, index):
    B, H, Hkv, Sq, Skv, P, D, window, sinks, ragged = shape
    a = call(dtype, *shape)
    if device.compute_units == 256:
        assert " | ".join(described(a)) == form
    rng = np.random.default_rng(index)
    lens = positions = None
    if ragged:
        lens = rng.integers(min(Sq, Skv), Skv + 1, B)
        positions = lens - Sq if Skv else rng.integers(-min(P, 50), 5, B)
    Call(device, dtype, B, H, Hkv, Sq, Skv, P, D, seed=index).both(lens=lens, positions=positions, offset=a.q_pos_offset, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [fa.F16, fa.BF16])
@pytest.mark.parametrize("index", range(len(CALLS_16)))
def test_16_bit(device, dtype, index):
    *shape, form = CALLS_16[index]
    check(device, dtype, shape, form, index)


@pytest.mark.parametrize("index", range(len(CALLS_F32)))
def test_f32(device, index):
    *shape, form = CALLS_F32[index]
    check(device, fa.F32, shape, form, index)
