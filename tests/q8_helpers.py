"""Uploads, read-backs and error bounds that the tests of the 8-bit cache share."""
import ctypes

import numpy as np

import floneum_amd as fa
from oracle import q8

HALF_STEP = {fa.F32: 2.0 ** -24, fa.F16: 2.0 ** -11, fa.BF16: 2.0 ** -8}


def rounded(x, dtype):
    """x (f32) rounded to dtype, as f32."""
    x = np.asarray(x, np.float32)
    if dtype == fa.F32:
        return x
    if dtype == fa.F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    return fa.bf16_bits_to_f32(fa.f32_to_bf16_bits(x))


def upload(device, x, dtype, order=None):
    """A tensor of x's shape; `order`: the order of its dimensions in memory (the others' strides follow)."""
    if order is None:
        return fa.Tensor.from_numpy(device, np.asarray(x, np.float32), dtype)
    t = fa.Tensor.from_numpy(device, np.ascontiguousarray(np.asarray(x, np.float32).transpose(order)), dtype)
    back = np.argsort(order)
    return fa.Tensor(t.buffer, dtype, [t.shape[i] for i in back], [t.strides[i] for i in back])


def spread(device, shape, dtype, steps, fill):
    """A tensor of `shape` whose strides are `steps` times a contiguous one's, in memory of value `fill` (a view that leaves gaps)."""
    whole = fa.Tensor.from_numpy(device, np.full([n * s for n, s in zip(shape, steps)], fill, np.float32), dtype)
    return whole, fa.Tensor(whole.buffer, dtype, shape, [st * s for st, s in zip(whole.strides, steps)])


def _bytes_to(device, array):
    a = np.ascontiguousarray(array)
    b = fa.Buffer(device, max(a.nbytes, 1))
    if a.nbytes:
        fa.check(fa.lib().fhip_memcpy_h2d(device.stream, ctypes.c_void_p(b.ptr), a.ctypes.data_as(ctypes.c_void_p), a.nbytes))
    return b


def _bytes_from(device, buffer, nbytes):
    a = np.empty(nbytes, np.uint8)
    if nbytes:
        fa.check(fa.lib().fhip_memcpy_d2h(device.stream, a.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(buffer.ptr), nbytes))
    return a


def upload_q8(device, codes, scales, fmt, block, first=0):
    """codes uint8 [B,H,rows,D], scales f32 [B,H,blocks]: a Q8Tensor (rows padded with zero bytes to 16)."""
    B, H, rows, D = codes.shape
    pitch = (D + 15) // 16 * 16
    padded = np.zeros((B, H, rows, pitch), np.uint8)
    padded[..., :D] = codes
    blocks = scales.shape[-1]
    return fa.Q8Tensor(_bytes_to(device, padded), _bytes_to(device, scales.astype(np.float32)), codes.shape, fmt, block,
                       (H * rows * pitch, rows * pitch, pitch), 0, (H * blocks, blocks), 0, first)


def download_q8(t):
    """(codes, scales) of a Q8Tensor that starts at its buffers' beginning."""
    B, H, rows, D = t.shape
    pitch, blocks = t.strides[2], t.scale_strides[1]
    assert t.offset == 0 and t.scale_offset == 0 and t.strides[1] == rows * pitch
    codes = _bytes_from(t.device, t.codes, B * H * rows * pitch).reshape(B, H, rows, pitch)
    scales = _bytes_from(t.device, t.scales, 4 * B * H * blocks).view(np.float32).reshape(B, H, blocks)
    return codes[..., :D], scales


def random_cache(rng, B, H, rows, D, fmt, block, std=1.0, first=0):
    """Codes and scales of N(0, std^2) rows."""
    codes = np.zeros((B, H, rows, D), np.uint8)
    scales = np.zeros((B, H, (first + rows + block - 1) // block if rows else 0), np.float32)
    x = rng.standard_normal((B, H, rows, D)).astype(np.float32) * np.float32(std)
    for b in range(B):
        for h in range(H):
            if block == 1 and rows:
                scales[b, h] = np.maximum(np.abs(x[b, h]).max(-1) * (np.float32(1) / np.float32(q8.LARGEST[fmt])), q8.LEAST_SCALE)
                codes[b, h] = q8.encode(x[b, h], scales[b, h][:, None], fmt)
            else:
                q8.append_rows(codes[b, h], scales[b, h], x[b, h], 0, fmt, block, first)
    return codes, scales


def attention_bound(out, mass, top, p, q, k, scale, v_scales, fmt, dtype, out_dtype):
    """How far an attention output may be from `out` (64 bits), element by element, from the roundings that the operator's description
    allows.  mass: sum of p |v|; top: the largest |score|; p: the probabilities; v_scales [B,Hkv,keys]."""
    n, D, eps = k.shape[2], q.shape[-1], 2.0 ** -24
    group = q.shape[1] // k.shape[1]
    reach = float(np.matmul(np.abs(q), np.repeat(np.abs(k), group, 1).swapaxes(-1, -2)).max()) * abs(scale) if n else 0.0
    # scores: f32 queries are two 11-bit terms (2^-22); a sum of D products; the product with the scales; the addition of the exponent
    score = (2.0 ** -22 * (dtype == fa.F32) + eps * (D + 8)) * reach + eps * (8 * top + 64)
    # probabilities: 11 bits, or two terms of them; exp2 to 2^-22
    rounding = (2.0 ** -22 if dtype == fa.F32 else 2.0 ** -11) + 2.0 ** -22
    sums = eps * (n / 32 + 256)
    # The products of a row's probabilities and scales are brought to f16 with the largest at 2^14 or more.  Below 2^-14 an f16 has a fixed step of
    # 2^-24, so the rounding of such a product (or of the second term of a larger one) is up to half of that, 2^-39 of the largest, and there are as
    # many as keys, each times a code.  16-bit queries may have a reference of up to 2^4 below the row's maximum, with the largest product that reference
    # allows still below 2^15: a row's largest is then at 2^10 or more, and half a step 2^-35 of it.
    weight = np.nan_to_num(np.nan_to_num(p) * np.repeat(v_scales, group, 1)[:, :, None, :]).max(-1, keepdims=True, initial=0.0)
    floor = 2.0 ** (-39 if dtype == fa.F32 else -35) * n * q8.LARGEST[fmt] * weight
    return HALF_STEP[out_dtype] * np.abs(out) + (2 * score + rounding + 2 * sums) * mass + floor + 1e-30
