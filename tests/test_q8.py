"""The 8-bit cache without a GPU: its CPU definition against first principles, the argument checks, the size query."""
import ctypes

import numpy as np
import pytest

import floneum_amd as fa
from oracle import q8

FAKE = 0x10000  # a non-null, 16-byte aligned stand-in for a device pointer; never dereferenced on the host


# ---- the definition ---------------------------------------------------------------------------------------------------

def test_e4m3_values():
    v = q8.E4M3_VALUES
    assert v[0x7E] == 448.0 and np.isnan(v[0x7F]) and np.isnan(v[0xFF]) and v[1] == 2.0 ** -9 and v[8] == 2.0 ** -6 and v[0x38] == 1.0
    assert np.array_equal(v[128:255], -v[:127]) and (np.diff(v[:127]) > 0).all()


@pytest.mark.parametrize("fmt", [q8.INT8, q8.E4M3])
def test_codes_are_the_nearest(fmt):
    rng = np.random.default_rng(1)
    values = np.unique(q8.code_values(np.arange(256, dtype=np.uint8), fmt)[[b for b in range(256) if b not in (127, 255) or fmt == q8.INT8]])
    values = values[np.abs(values) <= q8.LARGEST[fmt]]
    scale = np.float32(0.3)
    x = (rng.uniform(-1, 1, 4000) * q8.LARGEST[fmt] * float(scale)).astype(np.float32)
    got = q8.code_values(q8.encode(x, scale, fmt), fmt)
    nearest = values[np.abs(x[:, None].astype(np.float64) / np.float64(scale) - values[None, :]).argmin(1)]
    assert np.array_equal(np.abs(got), np.abs(nearest))
    # halfway: to the even code
    mid = (values[1:] + values[:-1]) / 2
    codes = q8.encode(mid.astype(np.float32), np.float32(1), fmt)
    assert (codes & 1 == 0).all()


@pytest.mark.parametrize("fmt", [q8.INT8, q8.E4M3])
def test_rows_that_join_a_block(fmt):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((40, 16)).astype(np.float32)
    whole, parts = (np.zeros((64, 16), np.uint8), np.zeros(2, np.float32)), (np.zeros((64, 16), np.uint8), np.zeros(2, np.float32))
    q8.append_rows(*whole, x, 3, fmt, 32)
    q8.append_rows(*parts, x[:10], 3, fmt, 32)
    for i in range(10, 40):
        q8.append_rows(*parts, x[i:i + 1], 3 + i, fmt, 32)
    assert np.array_equal(whole[1], parts[1])  # scales do not depend on how the rows came
    back = [q8.read_back(c, s, fmt, 32)[3:43] for c, s in (whole, parts)]
    step = (1.0 if fmt == q8.INT8 else 32.0) * whole[1].max()
    assert np.abs(back[0] - x).max() <= step / 2 * (1 + 1e-6) and np.abs(back[1] - x).max() <= 8 * step
    assert not whole[0][:3].any() and not whole[0][43:].any()


# ---- argument checks --------------------------------------------------------------------------------------------------

def t4(shape, ptr=FAKE, strides=None):
    st, acc = [], 1
    for n in reversed(shape):
        st.append(acc)
        acc *= n
    t = fa.CTensor4(ptr, 0)
    t.shape[:], t.stride[:] = shape, strides or list(reversed(st))
    return t


def t8(shape, block=1, fmt=0, first=0, codes=FAKE, scales=FAKE, **kw):
    B, H, rows, D = shape
    pitch, blocks = (D + 15) // 16 * 16, (first + rows + block - 1) // max(block, 1)
    t = fa.CQ8Tensor(codes, scales, 0, 0)
    t.shape[:], t.stride[:], t.scale_stride[:] = shape, (H * rows * pitch, rows * pitch, pitch), (H * blocks, blocks)
    t.block_tokens, t.first, t.format = block, first, fmt
    for name, value in kw.items():
        if name in ("stride", "scale_stride"):
            getattr(t, name)[:] = value
        else:
            setattr(t, name, value)
    return t


def attn(B=2, H=4, Hkv=2, Sq=1, Skv=300, D=64, dtype=fa.F16, k=None, v=None, **kw):
    a = fa.CQ8AttnArgs()
    a.q, a.out = t4([B, H, Sq, D]), t4([B, H, Sq, D])
    a.k, a.v = k or t8([B, Hkv, Skv, D]), v or t8([B, Hkv, Skv, D])
    a.dtype = a.out_dtype = dtype
    a.scale = 0.125
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def status(a):
    rc = fa.lib().fhip_q8_attention_validate(ctypes.byref(a))
    return rc, fa.lib().fhip_last_error().decode() if rc else ""


@pytest.mark.parametrize("dtype", [fa.F32, fa.F16, fa.BF16])
@pytest.mark.parametrize("D", [8, 64, 72, 80, 128, 200, 256])
def test_attention_accepts(dtype, D):
    assert status(attn(dtype=dtype, D=D))[0] == fa.OK
    assert status(attn(dtype=dtype, D=D, out_dtype=fa.F32))[0] == fa.OK


def mask(shape, ptr=FAKE):
    m = fa.CTensor2(ptr, 0)
    m.shape[:], m.stride[:] = shape, (shape[1], 1)
    return m


@pytest.mark.parametrize("change, code, text", [
    (dict(H=3), fa.ERR_INVALID_ARG, "must be divisible"),
    (dict(D=12), fa.ERR_UNSUPPORTED, "multiple of 8"),
    (dict(D=264), fa.ERR_UNSUPPORTED, "multiple of 8"),
    (dict(scale=float("nan")), fa.ERR_INVALID_ARG, "finite"),
    (dict(out_dtype=fa.BF16), fa.ERR_INVALID_ARG, "out_dtype"),
    (dict(dtype=7), fa.ERR_INVALID_ARG, "dtype"),
    (dict(out=t4([2, 4, 1, 32])), fa.ERR_INVALID_ARG, "output shape"),
    (dict(out=t4([2, 4, 1, 64], strides=[256, 0, 64, 1])), fa.ERR_INVALID_ARG, "overlapping"),
    (dict(q=t4([2, 4, 1, 64], ptr=0)), fa.ERR_INVALID_ARG, "device pointers"),
    (dict(k=t8([2, 2, 300, 64], codes=0)), fa.ERR_INVALID_ARG, "codes and scales"),
    (dict(k=t8([2, 2, 300, 64], scales=0)), fa.ERR_INVALID_ARG, "codes and scales"),
    (dict(k=t8([2, 2, 300, 64], fmt=1)), fa.ERR_INVALID_ARG, "differ in format"),
    (dict(k=t8([2, 2, 300, 64], fmt=2)), fa.ERR_INVALID_ARG, "format"),
    (dict(k=t8([2, 2, 300, 64], block=8)), fa.ERR_INVALID_ARG, "differ in format or block"),
    (dict(k=t8([2, 2, 300, 64], block=4)), fa.ERR_INVALID_ARG, "block_tokens"),
    (dict(k=t8([2, 2, 300, 64], block=8, first=8), v=t8([2, 2, 300, 64], block=8)), fa.ERR_INVALID_ARG, "first"),
    (dict(k=t8([2, 2, 299, 64])), fa.ERR_INVALID_ARG, "V shape"),
    (dict(k=t8([1, 2, 300, 64]), v=t8([1, 2, 300, 64])), fa.ERR_INVALID_ARG, "K shape"),
    (dict(k=t8([2, 2, 300, 64], offset=8)), fa.ERR_INVALID_ARG, "16 bytes"),
    (dict(k=t8([2, 2, 300, 64], stride=(1 << 20, 72, 64))), fa.ERR_INVALID_ARG, "16 bytes"),
    (dict(k=t8([2, 2, 300, 64], stride=(1 << 20, 1 << 16, 48))), fa.ERR_INVALID_ARG, "row stride"),
    (dict(k=t8([2, 2, 300, 64], stride=(1 << 20, 1 << 16, 1 << 26))), fa.ERR_INVALID_ARG, "row stride"),
    (dict(mask_kind=3), fa.ERR_INVALID_ARG, "mask_kind"),
    (dict(mask_kind=1), fa.ERR_INVALID_ARG, "QKMask shape"),
    (dict(mask_kind=1, mask=mask([2, 300])), fa.ERR_INVALID_ARG, "QKMask shape"),
    (dict(mask_kind=2, mask=mask([2, 299])), fa.ERR_INVALID_ARG, "BatchKeyMask shape"),
    (dict(mask_kind=2, mask=mask([2, 300], ptr=0)), fa.ERR_INVALID_ARG, "NULL"),
    (dict(mask=mask([1, 300])), fa.ERR_INVALID_ARG, "FHIP_MASK_NONE"),
    (dict(mask_kind=1, mask=mask([1, 300]), analytic=fa.CAnalyticMask(1, 1, 0, 0)), fa.ERR_INVALID_ARG, "exclusive"),
    (dict(analytic=fa.CAnalyticMask(1, 1, -1, 0)), fa.ERR_INVALID_ARG, "q_pos_offset"),
    (dict(analytic=fa.CAnalyticMask(1, 1, 0, -1)), fa.ERR_INVALID_ARG, "window"),
    (dict(analytic=fa.CAnalyticMask(1, 1, 1 << 62, 0)), fa.ERR_INVALID_ARG, "2\\^61"),
    (dict(q_positions=FAKE), fa.ERR_INVALID_ARG, "q_positions"),
    (dict(k=t8([2, 2, (1 << 31) - 4096, 64]), v=t8([2, 2, (1 << 31) - 4096, 64])), fa.ERR_UNSUPPORTED, "keys"),
])
def test_attention_refuses(change, code, text):
    rc, message = status(attn(**change))
    import re
    assert rc == code and re.search(text, message), message


def test_attention_without_elements():
    assert status(attn(B=0))[0] == fa.OK
    assert status(attn(Sq=0))[0] == fa.OK
    assert status(attn(Skv=0))[0] == fa.OK
    for a in (attn(B=0), attn(Sq=0), attn(Skv=0)):
        need = ctypes.c_size_t(7)
        assert fa.lib().fhip_q8_attention_workspace_bytes(ctypes.byref(a), 256, ctypes.byref(need)) == fa.OK and need.value == 0


def test_workspace_bytes():
    need = ctypes.c_size_t()
    one = attn(B=1, H=32, Hkv=8, Skv=4096, D=128)
    assert fa.lib().fhip_q8_attention_workspace_bytes(ctypes.byref(one), 256, ctypes.byref(need)) == fa.OK
    assert 0 < need.value < 64 << 20
    assert fa.lib().fhip_q8_attention_workspace_bytes(ctypes.byref(attn(Skv=100)), 256, ctypes.byref(need)) == fa.OK and need.value == 0
    assert fa.lib().fhip_q8_attention_workspace_bytes(ctypes.byref(attn(H=3)), 256, ctypes.byref(need)) == fa.ERR_INVALID_ARG
    assert fa.lib().fhip_q8_attention_workspace_bytes(ctypes.byref(one), 256, None) == fa.ERR_INVALID_ARG


# The append's checks come before anything that touches the device: a stand-in for a stream handle is never looked into.
def append(B=1, Hkv=2, n=3, D=64, rows=10, row=0, q=None, rope=None, **kw):
    a = fa.CQ8AppendArgs()
    a.k, a.v, a.row = t8([B, Hkv, rows, D]), t8([B, Hkv, rows, D]), row
    a.k_new, a.v_new = t4([B, Hkv, n, D]), t4([B, Hkv, n, D])
    a.in_dtype = fa.F16
    if q is not None:
        a.q, a.q_out, a.q_dtype, a.q_out_dtype = t4(q), t4(q), fa.F16, fa.F16
    if rope is not None:
        a.rope = ctypes.pointer(fa.CRopeTables(*rope))
    for name, value in kw.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("change, code, text", [
    (dict(row=8), fa.ERR_INVALID_ARG, "exceed"),
    (dict(row=1 << 40), fa.ERR_INVALID_ARG, "exceed"),
    (dict(n=0), fa.ERR_INVALID_ARG, "empty"),
    (dict(D=60), fa.ERR_UNSUPPORTED, "multiple of 8"),
    (dict(in_dtype=5), fa.ERR_INVALID_ARG, "dtype"),
    (dict(v_new=t4([1, 2, 2, 64])), fa.ERR_INVALID_ARG, "value shape"),
    (dict(k_new=t4([1, 3, 3, 64]), v_new=t4([1, 3, 3, 64])), fa.ERR_INVALID_ARG, "does not match the cache"),
    (dict(k_new=t4([1, 2, 3, 64], ptr=0)), fa.ERR_INVALID_ARG, "device pointers"),
    (dict(k=t8([1, 2, 10, 64], block=16)), fa.ERR_INVALID_ARG, "block_tokens"),
    (dict(k=t8([1, 2, 10, 64], stride=(1280, 0, 64))), fa.ERR_INVALID_ARG, "overlapping"),
    (dict(q=[1, 4, 2, 64]), fa.ERR_INVALID_ARG, "q shape"),
    (dict(q=[1, 4, 3, 64], q_out=t4([1, 4, 3, 32])), fa.ERR_INVALID_ARG, "q_out shape"),
    (dict(q=[1, 4, 3, 64], q_out=t4([1, 4, 3, 64], ptr=0)), fa.ERR_INVALID_ARG, "q_out"),
    (dict(q=[1, 4, 3, 64], q_dtype=9), fa.ERR_INVALID_ARG, "dtype"),
    (dict(rope=(FAKE, FAKE, 4, 2, 0)), fa.ERR_INVALID_ARG, "positions"),
    (dict(rope=(FAKE, 0, 4, 0, 0)), fa.ERR_INVALID_ARG, "NULL tables"),
    (dict(k_norm=ctypes.pointer(fa.CRmsNorm(0, 0, 0, 1e-6))), fa.ERR_INVALID_ARG, "rms norm"),
    (dict(n=1 << 29, rows=(1 << 31) - 100), fa.ERR_UNSUPPORTED, "2\\^30"),
])
def test_append_refuses(change, code, text):
    import re
    stream = ctypes.create_string_buffer(64)
    a = append(**change)
    rc = fa.lib().fhip_q8_append(ctypes.cast(stream, ctypes.c_void_p), ctypes.byref(a))
    message = fa.lib().fhip_last_error().decode()
    assert rc == code and re.search(text, message), message
    assert fa.lib().fhip_q8_append(None, ctypes.byref(a)) == fa.ERR_INVALID_ARG
    assert fa.lib().fhip_q8_append(ctypes.cast(stream, ctypes.c_void_p), None) == fa.ERR_INVALID_ARG


@pytest.mark.parametrize("row, out, dtype, text", [
    (8, t4([1, 2, 3, 64]), 0, "exceed"), (0, t4([1, 2, 3, 32]), 0, "output shape"), (0, t4([1, 2, 3, 64]), 4, "dtype"),
    (0, t4([1, 2, 3, 64], ptr=0), 0, "device pointer"), (0, t4([1, 2, 3, 64], strides=[384, 0, 64, 1]), 0, "overlapping"),
])
def test_dequantize_refuses(row, out, dtype, text):
    stream = ctypes.create_string_buffer(64)
    x = t8([1, 2, 10, 64])
    rc = fa.lib().fhip_q8_dequantize(ctypes.cast(stream, ctypes.c_void_p), ctypes.byref(x), row, None, ctypes.byref(out), dtype)
    assert rc == fa.ERR_INVALID_ARG and text in fa.lib().fhip_last_error().decode()


def test_cache_refuses():
    L, out = fa.lib(), ctypes.c_void_p()
    dev = ctypes.cast(ctypes.create_string_buffer(4096), ctypes.c_void_p)
    for fmt, block, rows in ((2, 1, 10), (0, 3, 10), (0, 0, 10), (0, 1, 0), (0, 1, 1 << 30)):
        assert L.fhip_q8_cache_create(dev, fmt, block, rows, ctypes.byref(out)) == fa.ERR_INVALID_ARG
    assert L.fhip_q8_cache_create(None, 0, 1, 10, ctypes.byref(out)) == fa.ERR_INVALID_ARG
    assert L.fhip_q8_cache_reset(None) == fa.ERR_INVALID_ARG and L.fhip_q8_cache_destroy(None) == fa.OK
    assert L.fhip_q8_cache_current_seq_len(None, None) == fa.ERR_INVALID_ARG


def test_struct_layout_matches_header():
    assert (ctypes.sizeof(fa.CQ8Tensor), ctypes.sizeof(fa.CQ8AppendArgs), ctypes.sizeof(fa.CQ8AttnArgs)) == (104, 528, 448)


def test_views():
    class Memory:
        device, ptr = None, FAKE
    x = fa.Q8Tensor(Memory(), Memory(), (2, 3, 100, 72), fa.Q8Format.INT8, 16)
    assert x.strides == (3 * 100 * 80, 100 * 80, 80) and x.scale_strides == (3 * 7, 7)
    y = x.narrow(2, 21, 50).narrow(0, 1, 1).narrow(1, 2, 1)
    assert y.shape == (1, 1, 50, 72) and y.first == 5 and y.offset == 24000 + 2 * 8000 + 21 * 80 and y.scale_offset == 21 + 14 + 1
    z = y.narrow(2, 12, 3)
    assert z.first == 1 and z.scale_offset == y.scale_offset + 1
    with pytest.raises(AssertionError):
        x.narrow(2, 60, 50)
