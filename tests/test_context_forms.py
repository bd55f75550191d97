"""The launches that the plan of attention over a context in two parts chooses, without a GPU."""
import pytest

import floneum_amd as fa
from context_forms import CALLS_16, CALLS_F32, described, forms
from test_context import FAKE, args


def call(dtype, B, H, Hkv, Sq, Skv, P, D, window, sinks, ragged):
    return args(B=B, H=H, Hkv=Hkv, Sq=Sq, Skv=Skv, P=P, D=D, dtype=dtype, out_dtype=dtype, window=window, sinks=sinks, scale=D ** -0.5,
                q_pos_offset=P if ragged or Skv == 0 else P + Skv - Sq, kv_lens=FAKE if ragged else None, q_positions=FAKE if ragged else None)


@pytest.mark.parametrize("dtype, calls", [(fa.F16, CALLS_16), (fa.BF16, CALLS_16), (fa.F32, CALLS_F32)])
def test_forms(dtype, calls):
    for *shape, form in calls:
        a = call(dtype, *shape)
        assert " | ".join(described(a)) == form, shape
        assert sum(f.rows for f in forms(a)) == shape[3]


@pytest.mark.parametrize("calls, launches", [
    (CALLS_16, ["128x2: ", "256x1: ", "128x1: ", "16 columns: ", "32 columns: "]), (CALLS_F32, ["64x2: ", "128x1: ", "128x2: ", "16 columns: "]),
])
def test_the_calls_reach_every_launch(calls, launches):
    """Rows of all sequences on the prefix with and without own keys beside them on tiles and in the kernel for few rows, in shares and whole; the last rows apart."""
    reached = {part for *_, form in calls for part in form.split(" | ")}
    for launch in launches:
        for part in ("own", "own /", "prefix", "prefix /"):
            assert launch + part in reached, (launch, part)
        if "columns" not in launch:
            for part in ("all prefix", "all prefix /", "all prefix /, own", "all prefix, own", "all prefix /, own /", "all prefix, own /"):
                assert launch + part in reached, (launch, part)
            assert any(r.startswith(launch + "all prefix /; ") for r in reached), launch
    assert sum(" | " in form for *_, form in calls) >= 10


@pytest.mark.parametrize("dtype", [fa.F16, fa.BF16])
@pytest.mark.parametrize("D", [64, 72, 96, 104, 128])
@pytest.mark.parametrize("scale", [1e-6, 0.1, 1.0, 1.5, 3.0, 1000.0])
def test_scales_of_prompts(dtype, D, scale):
    """Prompts of 16-bit tensors stay on the tiled kernel at every scale that it can form the scores with: all but, in bf16 at the widths of the kernel itself, such as
    would raise elements of Q beyond the type."""
    a = args(B=1, H=32, Hkv=8, Sq=8192, Skv=8192, D=D, dtype=dtype, out_dtype=dtype, window=4096, sinks=16, scale=scale)
    raises = dtype == fa.BF16 and D in (64, 96, 128) and scale * 1.4426950408889634 >= 2.0
    assert [bool(f.tiles) for f in forms(a)] == [not raises]
