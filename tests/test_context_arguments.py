"""Arguments of the Python mirror's attention over a context in two parts that are refused before anything runs (host only)."""
import pytest

import floneum_amd as fa
from test_context import FAKE, _Stub


def eight_bits(shape, device):
    memory = type("B", (), dict(ptr=FAKE, device=device))
    return fa.Q8Tensor(memory(), memory(), shape, fa.Q8Format.INT8, 1)


def test_parts_in_eight_bits():
    """Neither part may be an 8-bit cache's, the prefix as little as a sequence's own keys."""
    dev = object()
    q, k, p = _Stub((1, 2, 1, 64), device=dev), _Stub((1, 2, 9, 64), device=dev), _Stub((1, 2, 5, 64), device=dev)
    k8, p8 = eight_bits((1, 2, 9, 64), dev), eight_bits((1, 2, 5, 64), dev)
    for own, prefix in (((k8, k8), (p, p)), ((k, k8), None), ((k, k), (p8, p8)), ((k, k), (p, p8)), ((k, k), (p8, p))):
        with pytest.raises(fa.InvalidArgument, match="q's type"):
            q.flash_attention(*own, 1.0, sinks=1, prefix=prefix, analytic=(True, 0, 4))


@pytest.mark.parametrize("prefix", [(), ("keys",), ("keys", "values", "more"), 5])
def test_a_prefix_is_keys_and_values(prefix):
    dev = object()
    q, k = _Stub((1, 2, 1, 64), device=dev), _Stub((1, 2, 9, 64), device=dev)
    with pytest.raises(fa.InvalidArgument, match="keys and values"):
        q.flash_attention(k, k, 1.0, prefix=prefix)


class _Device:
    compute_units = 256


@pytest.mark.parametrize("sinks, analytic, name", [
    (1.5, (True, 0, 4), "sinks"), ("four", (True, 0, 4), "sinks"), (-1, (True, 0, 4), "sinks"), (1 << 64, (True, 0, 4), "sinks"), (-(1 << 70), (True, 0, 4), "sinks"),
    (1, (True, 0.5, 4), "q_pos_offset"), (1, (True, 1 << 64, 4), "q_pos_offset"), (1, (True, 0, 1 << 64), "window"), (1, (True, 0, 4.5), "window"),
])
def test_whole_numbers_of_64_bits(sinks, analytic, name):
    dev = _Device()
    q, k = _Stub((1, 2, 1, 64), device=dev), _Stub((1, 2, 9, 64), device=dev)
    with pytest.raises(fa.InvalidArgument, match=name):
        q.flash_attention(k, k, 1.0, sinks=sinks, out=_Stub((1, 2, 1, 64), device=dev), analytic=analytic)
