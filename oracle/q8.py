"""The 8-bit key / value cache on the CPU: codes, scales, appends and attention, element by element from their definitions
(test infrastructure only; the product never calls it)."""
import numpy as np

INT8, E4M3 = 0, 1
LARGEST = {INT8: 127.0, E4M3: 448.0}
LEAST_SCALE = np.float32(2.0 ** -100)


def _e4m3_table():
    v = np.empty(256)
    for bits in range(256):
        exponent, fraction = bits >> 3 & 15, bits & 7
        x = fraction * 2.0 ** -9 if exponent == 0 else (8 + fraction) * 2.0 ** (exponent - 10)
        if exponent == 15 and fraction == 7:
            x = np.nan
        v[bits] = -x if bits & 128 else x
    return v


E4M3_VALUES = _e4m3_table()


def code_values(codes, fmt):
    """What codes (uint8) stand for before their scale, in 64 bits."""
    return codes.view(np.int8).astype(np.float64) if fmt == INT8 else E4M3_VALUES[codes]


def encode(x, scale, fmt):
    """Codes (uint8) nearest to x / scale, ties to even.  x, scale f32.  The quotient in 64 bits is near enough: it is at least 2^-30 from a tie
    or on one."""
    y = np.asarray(x, np.float64) / np.asarray(scale, np.float64)
    bad = ~np.isfinite(y)
    y = np.where(bad, 0.0, y)
    if fmt == INT8:
        c = np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    else:
        e = np.maximum(np.frexp(y)[1] - 1, -6)
        step = np.ldexp(1.0, e - 3)
        v = np.minimum(np.abs(np.rint(y / step) * step), 448.0)
        positive = E4M3_VALUES[:127]
        c = np.searchsorted(positive, v).astype(np.uint8)
        assert np.array_equal(positive[c], v)
        c = c | np.where(np.signbit(y), 128, 0).astype(np.uint8)
    return np.where(bad, 0, c).astype(np.uint8)


def scale_of(x, fmt):
    """The f32 scale of the block whose new rows are x (any shape)."""
    top = np.max(np.abs(np.asarray(x, np.float32)))
    if not np.isfinite(top):
        return np.float32(np.nan)
    return max(np.float32(top) * (np.float32(1) / np.float32(LARGEST[fmt])), LEAST_SCALE)


def read_back(codes, scales, fmt, block, first=0):
    """f32 values of rows codes[..., rows, dim] with scales[..., blocks]."""
    at = (first + np.arange(codes.shape[-2])) // block
    with np.errstate(invalid="ignore"):
        return code_values(codes, fmt).astype(np.float32) * scales[..., at][..., None].astype(np.float32)


def append_rows(codes, scales, rows, place, fmt, block, first=0):
    """One (batch, head): f32 rows [n, dim] to `place` .. of codes [rows, dim] (uint8) / scales [blocks], in place.  Rows outside are left
    out."""
    n = min(len(rows), codes.shape[0] - place)
    if place < 0 or n <= 0:
        return
    rows = np.asarray(rows[:n], np.float32)
    for b in range((first + place) // block, (first + place + n - 1) // block + 1):
        lo, hi = max(place, b * block - first), min(place + n, (b + 1) * block - first)
        new = rows[lo - place:hi - place]
        s = scale_of(new, fmt)
        start = max(0, b * block - first)
        if start < place and lo == place:  # earlier rows of the block
            before = np.float32(scales[b])
            s = np.float32(np.nan) if np.isnan(s) or np.isnan(before) else max(s, before)
            if not np.isnan(s) and s != before:
                old = code_values(codes[start:place], fmt).astype(np.float32) * before
                codes[start:place] = encode(old, s, fmt)
        codes[lo:hi] = 0 if np.isnan(s) else encode(new, s, fmt)
        scales[b] = s


def rms_norm(x, weight, bias, eps, cast):
    """RMS norm in f32 with the squares added left to right, one rounding per operation; `cast` rounds to the tensor's type."""
    x, w = np.asarray(x, np.float32), np.asarray(weight, np.float32)
    ss = np.add.accumulate(x * x, axis=-1, dtype=np.float32)[..., -1:]
    n = x / np.sqrt(ss / np.float32(x.shape[-1]) + np.float32(eps)) * w
    return cast(n + np.asarray(bias, np.float32) if bias is not None else n)


def rope(x, cos, sin, interleaved=False):
    """x [..., rows, dim] rotated by cos / sin [rows, dim / 2], f32, one rounding per operation."""
    x, half = np.asarray(x, np.float32), x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    y0, y1 = a * cos - b * sin, b * cos + a * sin
    if not interleaved:
        return np.concatenate([y0, y1], -1)
    return np.stack([y0, y1], -1).reshape(x.shape)


def attention(q, k, v, scale, hidden=None, add=None):
    """softmax(q k^T scale + add, keys where `hidden` left out) v in 64 bits.  q [B,H,Sq,D], k, v [B,Hkv,Skv,D], hidden / add broadcast to
    [B,H,Sq,Skv].  Returns (out, p |v| summed, largest |score|, p): what errors are relative to."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    group = q.shape[1] // k.shape[1]
    k, v = np.repeat(k, group, 1), np.repeat(v, group, 1)
    s = np.matmul(q, k.swapaxes(-1, -2)) * scale
    if add is not None:
        s = s + add
    if hidden is not None:
        hidden = np.broadcast_to(hidden, s.shape)
        s = np.where(hidden, -np.inf, s)
    with np.errstate(invalid="ignore"):
        p = np.exp(s - s.max(-1, keepdims=True))
        p = p / p.sum(-1, keepdims=True)
        if hidden is not None:
            p = np.where(hidden & (~hidden).any(-1, keepdims=True), 0.0, p)
            seen = ~hidden.all((1, 2))[:, None, :, None]  # (rows that nobody sees may hold anything)
            v = np.where(seen, v, 0.0)
        out, mass = np.matmul(p, v), np.matmul(p, np.abs(v))
    finite = s[np.isfinite(s)]
    return out, mass, float(np.abs(finite).max()) if finite.size else 0.0, p
