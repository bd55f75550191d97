"""The workspace of attention over a context in two parts is bounded by what the chip holds at once, whatever a call's rows and keys (host only)."""
import ctypes

import numpy as np
import pytest

import floneum_amd as fa
from context_forms import forms
from test_context import FAKE, args


def need_of(a):
    need = ctypes.c_size_t()
    assert fa.lib().fhip_context_attention_workspace_bytes(ctypes.byref(a), 256, ctypes.byref(need)) == fa.OK
    return need.value


@pytest.mark.parametrize("dtype, Sq, Skv, window", [(fa.F16, 8192, 8192, 4096), (fa.F16, 32768, 131072, 0), (fa.F32, 32768, 131072, 0), (fa.BF16, 8192, 131072, 0)])
@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_prompts_that_the_tiled_kernels_refuse(dtype, Sq, Skv, window, scale):
    """Their rows fill the device by themselves: one share, no workspace, and not the kernel of a wavefront per row."""
    a = args(B=1, H=32, Hkv=8, Sq=Sq, Skv=Skv, D=128, dtype=dtype, out_dtype=dtype, window=window, sinks=4, scale=scale, q_pos_offset=Skv - Sq)
    assert need_of(a) == 0
    (f,) = forms(a)
    assert not f.any and not f.tiles and f.slots == 1


@pytest.mark.parametrize("columns", [16, 32])
def test_more_workgroups_than_a_launch_has(columns):
    """16-bit rows of more than 2^24 blocks of 16 columns: in blocks of 32 while these fit, then the kernel of a wavefront per row."""
    a = args(B=1, H=32, Hkv=32, Sq=(1 << 24) * columns // 32 + 32, Skv=64, D=64, dtype=fa.F16, out_dtype=fa.F16, scale=-0.1)
    (f,) = forms(a)
    assert (f.any, f.columns) == ((0, 32) if columns == 16 else (1, 0)), f


@pytest.mark.parametrize("kw, dtype, most", [
    (dict(B=64, H=32, Hkv=8, Skv=131072, D=128, kv_lens=FAKE, q_positions=FAKE), fa.F16, 5 << 20),   # one token of each sequence in a view of a whole cache
    (dict(B=64, H=32, Hkv=8, Skv=131072, D=128, kv_lens=FAKE, q_positions=FAKE), fa.F32, 5 << 20),
    (dict(B=16, H=32, Hkv=8, Skv=500, P=100000, D=128, window=1000, sinks=4, kv_lens=FAKE, q_positions=FAKE), fa.F32, 18 << 20),
])
def test_steps_in_a_long_view(kw, dtype, most):
    assert need_of(args(dtype=dtype, out_dtype=dtype, scale=0.1, **kw)) <= most


@pytest.mark.parametrize("dtype", [fa.F32, fa.F16, fa.BF16])
def test_workspaces_are_bounded(dtype):
    """Places of rows: two for each (a prefix and own keys in launches of their own), and beside them shares only as long as four rounds of 768 workgroups of 32 columns,
    for each of two jobs, or three of 256 workgroups of 256 rows are not filled."""
    rng = np.random.default_rng(5)

    def drawn(lo, hi):
        return int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))

    for _ in range(600):
        Hkv, G, D = drawn(1, 64), drawn(1, 40), 8 * drawn(1, 32)
        Skv, P = (drawn(1, 1 << 24) if rng.random() < 0.9 else 0 for _ in range(2))
        Sq = drawn(1, 1 << 15)
        B = drawn(1, max(1, min(1 << 12, ((1 << 27) - 1) // (Hkv * G * Sq))))
        rows = B * Hkv * G * Sq
        if rows >= 1 << 27:
            continue
        a = args(B=B, H=Hkv * G, Hkv=Hkv, Sq=Sq, Skv=Skv, P=P, D=D, dtype=dtype, out_dtype=dtype, window=drawn(1, 1 << 20) if rng.random() < 0.5 else 0,
                 sinks=drawn(1, 200), causal=1, q_pos_offset=drawn(1, 1 << 24), scale=0.1 if rng.random() < 0.5 else -0.1, kv_lens=FAKE if rng.random() < 0.5 else None,
                 q_positions=FAKE if rng.random() < 0.5 else None)
        assert need_of(a) <= 4 * (D + 4) * (2 * rows + 2 * 4 * 768 * 32 + 3 * 256 * 256), (B, Hkv, G, Sq, Skv, P, D)
