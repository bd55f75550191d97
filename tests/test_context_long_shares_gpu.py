"""Attention over a context in two parts in the kernel for few rows where its plan has fewer shares than its keys fill: the shares are longer then, and the kernel deals
them by what is visible.  Against the definition in 64 bits (context_helpers), sequence by sequence."""
import numpy as np
import pytest

import floneum_amd as fa
from context_forms import forms
from context_helpers import Call, definition, rounded, upload, visible
from test_context import FAKE, args

pytestmark = pytest.mark.gpu
TYPES = [fa.F32, fa.F16, fa.BF16]


def run(device, dtype, B, H, Hkv, Skv, P, D, lens, positions, offset, window, sinks, seqs, most):
    """One token per sequence; the sequences' own keys are one memory ([1, 1, Skv, D], broadcast).  Checks sequences `seqs`; most: shares of the longer part."""
    rng = np.random.default_rng(Skv + P)
    one = lambda *s: rounded(rng.standard_normal(s).astype(np.float32), dtype)  # noqa: E731
    q, k, v, pk, pv = one(B, H, 1, D), one(1, 1, Skv, D), one(1, 1, Skv, D), one(1, Hkv, P, D), one(1, Hkv, P, D)
    shared = [fa.Tensor(t.buffer, dtype, (B, Hkv, Skv, D), (0, 0, D, 1)) for t in (upload(device, x, dtype) for x in (k, v))]
    scale = float(np.float32(D ** -0.5))
    few = forms(args(B=B, H=H, Hkv=Hkv, Skv=Skv, P=P, D=D, dtype=dtype, out_dtype=dtype, window=window, sinks=sinks, scale=scale, q_pos_offset=offset, kv_lens=FAKE,
                     q_positions=FAKE))[0].few
    assert few and (device.compute_units != 256 or max(x.shares for x in few) <= most), few
    got = upload(device, q, dtype).flash_attention(*shared, scale, analytic=(True, offset, window), sinks=sinks,
                                                   prefix=(upload(device, pk, dtype), upload(device, pv, dtype)) if P else None,
                                                   kv_lens=fa.IntTensor(device, np.asarray(lens, np.int32)),
                                                   q_positions=fa.IntTensor(device, np.asarray(positions, np.int32)))
    got = np.asarray(got.to_numpy(), np.float64)
    for b in seqs:
        seen = visible(1, 1, Skv, P, lens=lens[b:b + 1], positions=positions[b:b + 1], offset=offset, window=window, sinks=sinks)
        wide = [np.broadcast_to(x, (1, Hkv, Skv, D)) for x in (k, v)]
        want, bound = definition(q[b:b + 1], *wide, pk[0], pv[0], scale, seen, dtype, dtype)
        assert (np.abs(got[b] - want[0]) <= bound[0]).all(), (b, lens[b], positions[b])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, H, Hkv, Skv, D", [(24, 32, 32, 9000, 64), (80, 32, 32, 3001, 128), (24, 16, 16, 7777, 136)])
def test_own_keys(device, dtype, B, H, Hkv, Skv, D):
    """Sequences of one key, of a few steps, of all keys and beyond, of none that counts as such."""
    rng = np.random.default_rng(B)
    lens = rng.integers(1, Skv + 1, B)
    lens[:6] = 1, Skv, 130, Skv - 1, Skv + 5, 700
    run(device, dtype, B, H, Hkv, Skv, 0, D, lens, np.minimum(lens, Skv) - 1, 0, 0, 0, (0, 1, 2, 3, 4, 5, B - 1), 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", [0, 300, 60000])
def test_windows_over_a_long_prefix(device, dtype, spread):
    """Sequences that stand beside each other see a few thousand keys of 60000, dealt to shares of single steps; where they stand all over the prefix each share is longer
    than the plan's."""
    B, H, Hkv, Skv, P, D, window, sinks = 128, 8, 8, 40, 60000, 64, 1000, 5
    rng = np.random.default_rng(3)
    lens = rng.integers(1, Skv + 1, B)
    positions = lens - 1 - rng.integers(0, spread + 1, B)
    positions[:3] = lens[0] - 1, lens[1] - 1 - spread, lens[2] - 1 - spread // 2
    run(device, dtype, B, H, Hkv, Skv, P, D, lens, positions, P, window, sinks, (0, 1, 2, B - 1), 64)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq, Skv, window", [(1100, 2500, 0), (1100, 2500, 1400), (2200, 2300, 0)])
def test_prompts(device, dtype, Sq, Skv, window):
    """Rows that the tiled kernels refuse (a negative scale) and that fill the device by themselves."""
    c = Call(device, dtype, 1, 4, 1, Sq, Skv, 70, 136, scale=-0.08, seed=Sq)
    a = args(B=1, H=4, Hkv=1, Sq=Sq, Skv=Skv, P=70, D=136, dtype=dtype, out_dtype=dtype, window=window, sinks=3, scale=c.scale, q_pos_offset=70 + Skv - Sq)
    (f,) = forms(a)
    assert f.few and not f.tiles and (device.compute_units != 256 or max(x.shares for x in f.few) <= 8)
    c.both(offset=70 + Skv - Sq, window=window, sinks=3)
