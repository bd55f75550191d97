"""Sizes at which calls of the 8-bit cache are refused, without a GPU: the checks come before anything that touches the device, so stand-ins
for handles and device pointers are never looked into."""
import ctypes

import pytest

import floneum_amd as fa
from test_q8 import FAKE, append, t4, t8  # noqa: F401


def call(function, *args):
    """(status, message) of a library call on a stand-in for a stream."""
    stream = ctypes.create_string_buffer(64)
    rc = getattr(fa.lib(), function)(ctypes.cast(stream, ctypes.c_void_p), *args)
    return rc, fa.lib().fhip_last_error().decode() if rc else ""


@pytest.mark.parametrize("lens", [None, FAKE])
@pytest.mark.parametrize("n", [1, 3])
def test_rope_tables_without_rows(lens, n):
    """Rows whose position the tables do not hold are left out with device lengths, but there has to be a row to read in their place."""
    rc, message = call("fhip_q8_append", ctypes.byref(append(n=n, rope=(FAKE, FAKE, 0, 0, 0), lens=lens)))
    assert rc == fa.ERR_INVALID_ARG and "tables" in message


@pytest.mark.parametrize("block", [1, 8, 16, 32, 64])
def test_longest_cache(block):
    """A cache slides through 2 * max_sequence_len rows in whole blocks and two blocks more, and every row's number has 31 bits."""
    longest = (1 << 30) - 128
    assert -(-2 * longest // block) * block + 2 * block < 1 << 31
    dev, out = ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p), ctypes.c_void_p()
    assert fa.lib().fhip_q8_cache_create(dev, 0, block, longest + 1, ctypes.byref(out)) == fa.ERR_INVALID_ARG and not out.value
    assert "2^30-128" in fa.lib().fhip_last_error().decode()


@pytest.mark.parametrize("heads, D", [(1 << 28, 64), ((1 << 31) // 9 + 1, 72), (1 << 26, 256), (1 << 30, 256)])
def test_reading_back_rows_of_too_many_heads(heads, D):
    """A launch numbers the pieces of eight elements in 31 bits and takes at least a row of all heads."""
    x, out = t8([1, heads, 1, D], stride=(0, 0, 256), scale_stride=(0, 0)), t4([1, heads, 1, D])
    rc, message = call("fhip_q8_dequantize", ctypes.byref(x), 0, None, ctypes.byref(out), 0)
    assert rc == fa.ERR_UNSUPPORTED and "2^34" in message


@pytest.mark.parametrize("missing", ["codes", "scales", "shape", "format", "block_tokens", "strides", "offset", "scale_strides", "scale_offset", "first"])
def test_parts_of_a_tensor_that_lacks_something(missing):
    class Memory:
        device, ptr = None, FAKE
    fa.lib()
    x = fa.Q8Tensor(Memory(), Memory(), (2, 3, 100, 72), fa.Q8Format.INT8, 16)
    delattr(x, missing)
    with pytest.raises(AttributeError, match=missing):
        x.narrow(2, 1, 2)


@pytest.mark.parametrize("with_native", [True, False])
def test_caches_of_two_devices(monkeypatch, with_native):
    """Keys and values of an append lie on one device, as everything else of a call."""
    class Memory:
        def __init__(self, device):
            self.device, self.ptr = device, FAKE
    fa.lib()
    if not with_native:
        monkeypatch.setattr(fa, "_native", None)
    here, there = object(), object()
    keys, values = (fa.Q8Tensor(Memory(d), Memory(d), (1, 2, 10, 64), fa.Q8Format.INT8, 1) for d in (here, there))
    rows = fa.Tensor(Memory(here), fa.F16, (1, 2, 3, 64))
    with pytest.raises(AssertionError, match="different devices"):
        keys.append(values, rows, rows)


def test_both_caches_are_called_alike():
    """A program changes to the 8-bit cache by the class it creates: the steps of both take the same arguments."""
    import inspect
    for name in ("append", "append_rope", "qkv_rope_append"):
        wide, narrow = (list(inspect.signature(getattr(c, name)).parameters) for c in (fa.KvCache, fa.Q8KvCache))
        assert wide == narrow, name
