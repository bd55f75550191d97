"""Attention over a context in two parts without a GPU: the definition's mask, the argument checks, the size query."""
import ctypes
import re

import numpy as np
import pytest

import floneum_amd as fa
from context_helpers import visible

FAKE = 0x10000  # a non-null, 16-byte aligned stand-in for a device pointer; never dereferenced on the host


def t4(shape, ptr=FAKE, strides=None):
    st, acc = [], 1
    for n in reversed(shape):
        st.append(acc)
        acc *= n
    t = fa.CTensor4(ptr, 0)
    t.shape[:], t.stride[:] = shape, strides or st[::-1]
    return t


def args(B=2, H=4, Hkv=2, Sq=1, Skv=300, P=0, D=64, **kw):
    a = fa.CContextAttnArgs()
    a.q, a.out, a.k, a.v = t4([B, H, Sq, D]), t4([B, H, Sq, D]), t4([B, Hkv, Skv, D]), t4([B, Hkv, Skv, D])
    if P:
        a.prefix_k, a.prefix_v = t4([1, Hkv, P, D]), t4([1, Hkv, P, D])
    a.dtype = a.out_dtype = fa.F16
    a.scale, a.causal = 0.125, 1
    for name, x in kw.items():
        setattr(a, name, x)
    return a


def status(a):
    rc = fa.lib().fhip_context_attention_validate(ctypes.byref(a))
    return rc, fa.lib().fhip_last_error().decode() if rc else ""


def test_visible_is_the_rule():
    seen = visible(2, 3, 6, 4, lens=[6, 2], positions=[0, -2], offset=7, window=3, sinks=2)
    for b, (length, start) in enumerate(((6, 7), (2, 5))):
        for i in range(3):
            for j in range(10):
                p = start + i
                assert seen[b, i, j] == (j < 4 + length and j <= p and (j + 3 > p or j < 2))


@pytest.mark.parametrize("change, code, text", [
    (dict(H=3), fa.ERR_INVALID_ARG, "must be divisible"),
    (dict(D=520), fa.ERR_UNSUPPORTED, "head_dim"),
    (dict(scale=float("inf")), fa.ERR_INVALID_ARG, "finite"),
    (dict(out_dtype=fa.BF16), fa.ERR_INVALID_ARG, "out_dtype"),
    (dict(dtype=3), fa.ERR_INVALID_ARG, "dtype"),
    (dict(out=t4([2, 4, 1, 32])), fa.ERR_INVALID_ARG, "output shape"),
    (dict(out=t4([2, 4, 1, 64], strides=[256, 0, 64, 1])), fa.ERR_INVALID_ARG, "overlapping"),
    (dict(q=t4([2, 4, 1, 64], ptr=0)), fa.ERR_INVALID_ARG, "device pointers"),
    (dict(k=t4([2, 2, 300, 64], ptr=0)), fa.ERR_INVALID_ARG, "device pointers"),
    (dict(v=t4([2, 2, 299, 64])), fa.ERR_INVALID_ARG, "V shape"),
    (dict(k=t4([1, 2, 300, 64]), v=t4([1, 2, 300, 64])), fa.ERR_INVALID_ARG, "K shape"),
    (dict(prefix_k=t4([1, 2, 50, 64])), fa.ERR_INVALID_ARG, "prefix V shape"),
    (dict(prefix_k=t4([2, 2, 50, 64]), prefix_v=t4([2, 2, 50, 64])), fa.ERR_INVALID_ARG, "prefix shape"),
    (dict(prefix_k=t4([1, 4, 50, 64]), prefix_v=t4([1, 4, 50, 64])), fa.ERR_INVALID_ARG, "prefix shape"),
    (dict(prefix_k=t4([1, 2, 50, 32]), prefix_v=t4([1, 2, 50, 32])), fa.ERR_INVALID_ARG, "prefix shape"),
    (dict(prefix_k=t4([1, 2, 50, 64], ptr=0), prefix_v=t4([1, 2, 50, 64])), fa.ERR_INVALID_ARG, "prefix_k"),
    (dict(q_pos_offset=-1), fa.ERR_INVALID_ARG, "q_pos_offset"),
    (dict(window=-1), fa.ERR_INVALID_ARG, "window"),
    (dict(sinks=-1), fa.ERR_INVALID_ARG, "sinks"),
    (dict(q_pos_offset=1 << 62), fa.ERR_INVALID_ARG, "2\\^61"),
    (dict(window=1 << 62), fa.ERR_INVALID_ARG, "2\\^61"),
    (dict(causal=0, q_positions=FAKE), fa.ERR_INVALID_ARG, "q_positions"),
    (dict(Skv=(1 << 31) - 4096), fa.ERR_UNSUPPORTED, "keys"),
    (dict(Skv=(1 << 30), P=(1 << 30)), fa.ERR_UNSUPPORTED, "keys"),
    (dict(B=1 << 15, H=1 << 10, Hkv=1, Sq=1 << 7), fa.ERR_UNSUPPORTED, "query rows"),
    (dict(Sq=1 << 31), fa.ERR_INVALID_ARG, "2\\^31-1"),
])
def test_refusals(change, code, text):
    rc, message = status(args(**change))
    assert rc == code and re.search(text, message), message


def test_null_arguments():
    L = fa.lib()
    need = ctypes.c_size_t()
    assert L.fhip_context_attention_validate(None) == fa.ERR_INVALID_ARG
    assert L.fhip_context_attention(None, ctypes.byref(args())) == fa.ERR_INVALID_ARG
    assert L.fhip_context_attention_workspace_bytes(ctypes.byref(args()), 256, None) == fa.ERR_INVALID_ARG
    assert L.fhip_context_attention_workspace_bytes(None, 256, ctypes.byref(need)) == fa.ERR_INVALID_ARG
    assert L.fhip_context_attention_workspace_bytes(ctypes.byref(args(H=3)), 256, ctypes.byref(need)) == fa.ERR_INVALID_ARG


def test_tensors_without_elements():
    for a in (args(B=0), args(Sq=0), args(Skv=0), args(P=1, Skv=0), args(B=0, k=t4([0, 2, 300, 64], ptr=0), v=t4([0, 2, 300, 64], ptr=0))):
        assert status(a) == (fa.OK, "")
    for a in (args(B=0), args(Sq=0), args(Skv=0)):
        need = ctypes.c_size_t(7)
        assert fa.lib().fhip_context_attention_workspace_bytes(ctypes.byref(a), 256, ctypes.byref(need)) == fa.OK and need.value == 0


def test_accepted():
    for a in (args(P=5), args(window=10, sinks=4), args(sinks=1 << 40), args(window=1 << 60, q_pos_offset=1 << 60), args(causal=0), args(D=7, P=9),
              args(out_dtype=fa.F32), args(dtype=fa.F32, out_dtype=fa.F32), args(scale=-1.0), args(q_positions=FAKE, kv_lens=FAKE)):
        assert status(a) == (fa.OK, "")


class _Stub:
    """A tensor as the argument checks of the mirror see it."""

    def __new__(cls, shape, dtype=fa.F16, device=None):
        buffer = type("B", (), dict(ptr=FAKE, device=device))()
        return fa.Tensor(buffer, dtype, shape)


def test_python_refusals():
    dev = object()
    q, k = _Stub((1, 2, 1, 64), device=dev), _Stub((1, 2, 9, 64), device=dev)
    p = _Stub((1, 2, 5, 64), device=dev)
    other = _Stub((1, 2, 5, 64), device=object())
    wide = _Stub((1, 2, 5, 64), fa.F32, dev)
    mask = _Stub((1, 9), device=dev)
    for kw, error in ((dict(sinks=1, mask=(mask, fa.MaskKind.QKMask)), fa.InvalidArgument), (dict(prefix=(p, other)), AssertionError),
                      (dict(prefix=(p, wide)), fa.InvalidArgument), (dict(sinks=1, force_kernel=1), fa.InvalidArgument),
                      (dict(prefix=(p, _Stub((2, 5, 64), device=dev))), fa.InvalidArgument),
                      (dict(sinks=1, out=_Stub((1, 2, 1, 64), device=dev), out_dtype=fa.F32), fa.InvalidArgument),
                      (dict(sinks=1, out=_Stub((1, 2, 1, 64), device=object())), AssertionError)):
        with pytest.raises(error):
            q.flash_attention(k, k, 1.0, **kw)


def test_python_lengths():
    dev = object()
    q, k = _Stub((2, 2, 1, 64), device=dev), _Stub((2, 2, 9, 64), device=dev)

    def lens(n, device, dtype="i32"):
        return type("L", (), dict(dtype=dtype, shape=(n,), offset=0, buffer=type("B", (), dict(ptr=FAKE, device=device))()))()

    for kw, error in ((dict(kv_lens=lens(2, object())), AssertionError), (dict(q_positions=lens(2, object())), AssertionError),
                      (dict(kv_lens=lens(3, dev)), fa.InvalidArgument), (dict(q_positions=lens(2, dev, "f32")), fa.InvalidArgument),
                      (dict(kv_lens=np.zeros(2, np.int32)), fa.InvalidArgument)):
        with pytest.raises(error):
            q.flash_attention(k, k, 1.0, sinks=1, analytic=(True, 0, 4), **kw)


@pytest.mark.parametrize("dtype", [fa.F32, fa.F16, fa.BF16])
def test_workspaces_of_any_call(dtype):
    """The size query answers for every shape within the limits, and asks for no more than a share of the keys that a call reads: a row's place holds
    D + 4 floats and stands for 64 keys of D elements and more."""
    rng = np.random.default_rng(3)
    need = ctypes.c_size_t()

    def drawn(lo, hi):
        return int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))

    for _ in range(400):
        Hkv, G, D = drawn(1, 64), drawn(1, 40), 8 * drawn(1, 32)
        Skv, P = (drawn(1, 1 << 24) if rng.random() < 0.9 else 0 for _ in range(2))
        Sq = drawn(1, 1 << 16)
        B = drawn(1, max(1, min(1 << 16, ((1 << 31) - 1) // (Hkv * G * Sq))))
        if B * Hkv * G * Sq >= 1 << 31:
            continue
        a = args(B=B, H=Hkv * G, Hkv=Hkv, Sq=Sq, Skv=Skv, P=P, D=D, dtype=dtype, out_dtype=dtype, window=drawn(1, 1 << 20) if rng.random() < 0.5 else 0,
                 sinks=drawn(1, 200), causal=1, q_pos_offset=drawn(1, 1 << 24), kv_lens=FAKE if rng.random() < 0.5 else None)
        assert fa.lib().fhip_context_attention_workspace_bytes(ctypes.byref(a), 256, ctypes.byref(need)) == fa.OK
        assert need.value <= B * Hkv * G * Sq * 4 * (D + 4) * (2 + (Skv + 63) // 64 + (P + 63) // 64)


def test_limits_of_rows():
    """2^31 - 4097 rows at most: a workgroup's last row is counted in 32 bits."""
    top = (1 << 31) - 4097
    assert status(args(B=1, H=1, Hkv=1, Sq=top, D=8)) == (fa.OK, "")
    for a in (args(B=1, H=1, Hkv=1, Sq=top + 1, D=8), args(B=1 << 10, H=1 << 10, Hkv=1, Sq=1 << 11, D=8)):
        rc, message = status(a)
        assert rc == fa.ERR_UNSUPPORTED and "query rows" in message
    need = ctypes.c_size_t()
    for Skv, P in ((1, 0), (1, 1), (0, 100), (100000, 5)):  # (rows times shares beyond what a launch takes: another kernel's)
        for B, Sq in ((1, top), (top // 64, 64), (top, 1)):
            a = args(B=B, H=1, Hkv=1, Sq=Sq, Skv=Skv, P=P, D=8)
            assert fa.lib().fhip_context_attention_workspace_bytes(ctypes.byref(a), 256, ctypes.byref(need)) == fa.OK
