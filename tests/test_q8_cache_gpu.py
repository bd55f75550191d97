"""Rows coded into the 8-bit cache and read back on the GPU, bit for bit against the definition (oracle/q8.py)."""
import ctypes

import numpy as np
import pytest

import floneum_amd as fa
from oracle import q8
from q8_helpers import download_q8, random_cache, rounded, spread, upload, upload_q8

pytestmark = pytest.mark.gpu

F32, F16, BF16 = fa.F32, fa.F16, fa.BF16
INT8, E4M3 = q8.INT8, q8.E4M3


def normals(rng, shape, dtype, std=1.0):
    return rounded(rng.standard_normal(shape).astype(np.float32) * np.float32(std), dtype)


def expected(codes, scales, rows, places, fmt, block, first=0, counts=None):
    """codes / scales after rows [B,H,n,D] go to places[b] .. ."""
    codes, scales = codes.copy(), scales.copy()
    for b in range(codes.shape[0]):
        n = rows.shape[2] if counts is None else min(max(counts[b], 0), rows.shape[2])
        for h in range(codes.shape[1]):
            q8.append_rows(codes[b, h], scales[b, h], rows[b, h, :n], places[b], fmt, block, first)
    return codes, scales


def same_codes(got, want, fmt):
    if fmt == E4M3:  # the sign of a zero does not matter
        got, want = got & np.where(got & 127, 255, 127), want & np.where(want & 127, 255, 127)
    return np.array_equal(got, want)


def same(t, codes, scales, fmt):
    got = download_q8(t)
    assert np.array_equal(got[1], scales, equal_nan=True), np.argwhere(~((got[1] == scales) | np.isnan(scales)))[:5]
    assert same_codes(got[0], codes, fmt), np.argwhere(got[0] != codes)[:5]


# ---- coding -------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("block", [1, 8, 16, 32, 64])
@pytest.mark.parametrize("dtype, D", [(F32, 8), (F16, 64), (BF16, 72), (F32, 80), (F16, 128), (F32, 136), (BF16, 200), (F16, 256)])
def test_rows_into_an_empty_cache(device, fmt, block, dtype, D):
    rng = np.random.default_rng(D * 100 + block)
    B, H, n, rows = 2, 3, 77, 130
    k, v = normals(rng, (B, H, n, D), dtype), normals(rng, (B, H, n, D), dtype, 30.0)
    k8, v8 = (fa.Q8Tensor.empty(device, (B, H, rows, D), fa.Q8Format(fmt), block) for _ in range(2))
    k8.append(v8, upload(device, k, dtype), upload(device, v, dtype), 5)
    empty = np.zeros((B, H, rows, D), np.uint8), np.zeros((B, H, -(-rows // block)), np.float32)
    same(k8, *expected(*empty, k, [5] * B, fmt, block), fmt)
    same(v8, *expected(*empty, v, [5] * B, fmt, block), fmt)
    want = q8.read_back(*download_q8(v8), fmt, block)
    for out in (F32, F16, BF16):
        assert np.array_equal(np.asarray(v8.dequantize(out).to_numpy(), np.float32), rounded(want, out))


@pytest.mark.parametrize("fmt", [INT8, E4M3])
def test_codes_next_to_a_border(device, fmt):
    """Quotients on and next to the middle between two codes, for scales that are and are not powers of two."""
    rng = np.random.default_rng(3)
    values = np.unique(np.abs(q8.code_values(np.array([b for b in range(256) if b & 127 != 127], np.uint8), fmt)))
    values = values[values <= q8.LARGEST[fmt]]
    mid = (values[1:] + values[:-1]) / 2
    rows = []
    for top in (np.float32(q8.LARGEST[fmt]), np.float32(3.0), np.float32(1.0) / 3, np.float32(7e-20), np.float32(5e30)):
        s = q8.scale_of(np.array([top]), fmt)
        m = (mid * np.float64(s)).astype(np.float32)
        for x in (m, np.nextafter(m, np.float32(0)), np.nextafter(m, top)):
            x = np.concatenate([x * rng.choice([-1, 1], x.size).astype(np.float32)])[:255]
            rows.append(np.concatenate([[top], np.minimum(np.abs(x), top) * np.sign(x), np.zeros(255 - x.size)]).astype(np.float32))
    x = np.stack(rows)[None, None]
    k8, v8 = (fa.Q8Tensor.empty(device, (1, 1, x.shape[2], 256), fa.Q8Format(fmt), 1) for _ in range(2))
    k8.append(v8, upload(device, x, F32), upload(device, -x, F32))
    empty = np.zeros((1, 1, x.shape[2], 256), np.uint8), np.zeros((1, 1, x.shape[2]), np.float32)
    same(k8, *expected(*empty, x, [0], fmt, 1), fmt)
    same(v8, *expected(*empty, -x, [0], fmt, 1), fmt)


@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("block", [1, 8, 64])
def test_values_without_a_code(device, fmt, block):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((1, 2, 200, 64)).astype(np.float32)
    x[0, 0, 3] = 0.0                    # a row of zeros
    x[0, 0, 70, 5] = np.nan
    x[0, 1, 9, 63] = np.inf
    x[0, 1, 140, 0] = -np.inf
    x[0, 1, 64:128] = 1e-45             # below the least scale
    x[0, 0, 130:140] = 3e38
    k8, v8 = (fa.Q8Tensor.empty(device, (1, 2, 200, 64), fa.Q8Format(fmt), block) for _ in range(2))
    k8.append(v8, upload(device, x, F32), upload(device, x, F32))
    empty = np.zeros((1, 2, 200, 64), np.uint8), np.zeros((1, 2, -(-200 // block)), np.float32)
    codes, scales = expected(*empty, x, [0], fmt, block)
    same(k8, codes, scales, fmt)
    same(v8, codes, scales, fmt)
    back = k8.dequantize().to_numpy()
    assert np.array_equal(back, q8.read_back(codes, scales, fmt, block), equal_nan=True)
    assert np.isnan(back[0, 0, 70]).all() and not np.isnan(back[0, 0, :64]).any()


@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("block", [1, 8, 32, 64])
@pytest.mark.parametrize("D", [64, 96, 256])
def test_token_by_token(device, fmt, block, D):
    """Single rows into blocks that are partly filled: scales grow, earlier rows are coded again."""
    rng = np.random.default_rng(block + D)
    B, H, rows = 2, 2, 70
    x = normals(rng, (2, B, H, rows, D), F32) * np.linspace(0.5, 2, rows, dtype=np.float32)[:, None]
    k8, v8 = (fa.Q8Tensor.empty(device, (B, H, rows, D), fa.Q8Format(fmt), block) for _ in range(2))
    state = [(np.zeros((B, H, rows, D), np.uint8), np.zeros((B, H, -(-rows // block)), np.float32)) for _ in range(2)]
    at = 0
    for n in [1, 1, 3, 1, 10, 1, 1, 20, 1, 1, 1, 25, 1, 1, 2]:
        new = x[:, :, :, at:at + n]
        k8.append(v8, upload(device, new[0], F32), upload(device, new[1], F32), at)
        state = [expected(*s, new[i], [at] * B, fmt, block) for i, s in enumerate(state)]
        at += n
    assert at == rows
    same(k8, *state[0], fmt)
    same(v8, *state[1], fmt)


@pytest.mark.parametrize("block", [1, 8, 64])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_sequences_of_their_own_lengths(device, block, n):
    """Device lens and counts: places that differ by sequence, rows that are left out, memory behind them as it was."""
    rng = np.random.default_rng(block * n)
    B, H, rows, D = 6, 2, 150, 64
    lens, counts = [0, 7, 64, 149, 200, -3], [n, 0, n + 5, n, n, n]
    first = 0 if block == 1 else 3
    state = [random_cache(rng, B, H, rows, D, INT8, block, first=first) for _ in range(2)]
    k8, v8 = (upload_q8(device, *s, fa.Q8Format.INT8, block, first) for s in state)
    k, v = normals(rng, (B, H, n, D), F16), normals(rng, (B, H, n, D), F16, 3.0)
    q = normals(rng, (B, 4, n, D), F16)
    rope = fa.RopeCache(D, 160, 10000.0, device)
    q_out = upload(device, np.full((B, 4, n, D), 5.0), F16)
    k8.append(v8, upload(device, k, F16), upload(device, v, F16), 1, lens=fa.IntTensor(device, lens), counts=fa.IntTensor(device, counts),
              rope=rope, start_pos=2, q=upload(device, q, F16), q_out=q_out)
    got_q = q_out.to_numpy().astype(np.float32)
    want = [(c.copy(), s.copy()) for c, s in state]
    for b in range(B):
        place = 1 + lens[b]
        m = max(0, min(counts[b], n, rows - place, 160 - (2 + lens[b]))) if place >= 0 and lens[b] + 2 >= 0 else 0
        if m:
            cos, sin = (t[2 + lens[b]:2 + lens[b] + m] for t in (rope.cos_host, rope.sin_host))
            for h in range(H):
                q8.append_rows(want[0][0][b, h], want[0][1][b, h], q8.rope(k[b, h, :m], cos, sin), place, INT8, block, first)
                q8.append_rows(want[1][0][b, h], want[1][1][b, h], v[b, h, :m], place, INT8, block, first)
            assert np.array_equal(got_q[b, :, :m], rounded(q8.rope(q[b, :, :m], cos, sin), F16))
        assert (got_q[b, :, m:] == 5.0).all()
    same(k8, *want[0], INT8)
    same(v8, *want[1], INT8)


# ---- norm, rotation, layouts -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype, D, block, n", [(F32, 64, 1, 9), (F16, 128, 1, 50), (BF16, 256, 32, 21), (F16, 80, 16, 33), (BF16, 72, 1, 4),
                                                (F32, 200, 8, 3), (F16, 64, 64, 70)])
def test_norm_and_rotation(device, dtype, D, block, n, normed, interleaved):
    """Keys are the f32 values that the wide cache's call rounds to its type, q is that call's q, bit for bit."""
    rng = np.random.default_rng(D + n)
    B, H, Hkv, fmt = 2, 4, 2, INT8 if block == 1 else E4M3
    q, k, v = (normals(rng, (B, h, n, D), dtype) for h in (H, Hkv, Hkv))
    rope = fa.RopeCache(D, 100, 10000.0, device)
    weight, bias = rng.normal(1, 0.3, (2, D)).astype(np.float32), rng.normal(0, 0.1, D).astype(np.float32)
    norms = [fa.RmsNorm(weight[0], None, 1e-6, F32, device), fa.RmsNorm(weight[1], bias, 1e-6, BF16, device)] if normed else [None, None]
    # projections as a model holds them, [batch, rows, heads, head_dim]
    tq, tk, tv = (upload(device, x, dtype, (0, 2, 1, 3)) for x in (q, k, v))
    k8, v8 = (fa.Q8Tensor.empty(device, (B, Hkv, 100, D), fa.Q8Format(fmt), block) for _ in range(2))
    got = k8.append(v8, tk, tv, 11, rope=rope, start_pos=13, interleaved=interleaved, k_norm=norms[1], q=tq, q_norm=norms[0], q_out_dtype=F32)
    wide = fa.KvCache(2, 100, F32, device)
    want_q, wide_k, _ = wide.qkv_rope_append(rope, tq, tk, tv, 13, interleaved, norms[0], norms[1], F32)
    assert np.array_equal(got.to_numpy(), want_q.to_numpy())
    keys = wide_k.to_numpy()
    cast = lambda x: rounded(x, dtype)  # noqa: E731
    plain = q8.rms_norm(k, rounded(weight[1], BF16), rounded(bias, BF16), 1e-6, cast) if normed else k
    assert np.array_equal(keys, q8.rope(plain, rope.cos_host[13:13 + n], rope.sin_host[13:13 + n], interleaved))
    empty = np.zeros((B, Hkv, 100, D), np.uint8), np.zeros((B, Hkv, -(-100 // block)), np.float32)
    same(k8, *expected(*empty, keys, [11] * B, fmt, block), fmt)
    same(v8, *expected(*empty, v, [11] * B, fmt, block), fmt)


def test_norm_without_rotation(device):
    rng = np.random.default_rng(8)
    k, v, q = normals(rng, (1, 2, 6, 128), F16), normals(rng, (1, 2, 6, 128), F16), normals(rng, (1, 4, 6, 128), F16)
    weight = rng.normal(1, 0.3, 128).astype(np.float32)
    norm = fa.RmsNorm(weight, None, 1e-5, F32, device)
    k8, v8 = (fa.Q8Tensor.empty(device, (1, 2, 6, 128)) for _ in range(2))
    q_out = k8.append(v8, upload(device, k, F16), upload(device, v, F16), k_norm=norm, q=upload(device, q, F16), q_norm=norm)
    cast = lambda x: rounded(x, F16)  # noqa: E731
    assert np.array_equal(q_out.to_numpy().astype(np.float32), q8.rms_norm(q, weight, None, 1e-5, cast))
    empty = np.zeros((1, 2, 6, 128), np.uint8), np.zeros((1, 2, 6), np.float32)
    same(k8, *expected(*empty, q8.rms_norm(k, weight, None, 1e-5, cast), [0], INT8, 1), INT8)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_strided_rows(device, dtype):
    """Sources and destinations with gaps between all elements, q rotated in place, a batch read with stride 0."""
    rng = np.random.default_rng(9)
    B, H, n, D = 2, 2, 7, 64
    x = normals(rng, (B, H, n, D), dtype)
    whole = normals(rng, (B * 2, H * 3, n * 2, D * 3), dtype)
    whole[::2, ::3, ::2, ::3] = x
    base = upload(device, whole, dtype)
    t = fa.Tensor(base.buffer, dtype, (B, H, n, D), [s * m for s, m in zip(base.strides, (2, 3, 2, 3))])
    rope = fa.RopeCache(D, 20, 10000.0, device)
    k8, v8 = (fa.Q8Tensor.empty(device, (B, H, n, D), fa.Q8Format.E4M3, 8) for _ in range(2))
    assert k8.append(v8, t, t, rope=rope, q=t, q_out=t) is t
    turned = q8.rope(x, rope.cos_host[:n], rope.sin_host[:n])
    whole[::2, ::3, ::2, ::3] = rounded(turned, dtype)
    assert np.array_equal(np.asarray(base.to_numpy(), np.float32), whole)
    empty = np.zeros((B, H, n, D), np.uint8), np.zeros((B, H, 1), np.float32)
    # (q is turned in place by the launch that also reads it as keys: those cannot be checked)
    one = upload(device, x[:1], dtype).broadcast_to((B, H, n, D))
    k8.append(v8, one, one)
    state = expected(*empty, np.repeat(x[:1], B, 0), [0] * B, E4M3, 8)
    same(k8, *state, E4M3)
    memory, out = spread(device, (B, H, n, D), dtype, (1, 2, 3, 2), 9.0)
    v8.dequantize(out=out)
    host = np.full(memory.shape, 9.0, np.float32)
    host[:, ::2, ::3, ::2] = rounded(q8.read_back(*state, E4M3, 8), dtype)
    assert np.array_equal(np.asarray(memory.to_numpy(), np.float32), host)


# ---- reading back ------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("block, D, rows", [(1, 128, 301), (16, 72, 50), (64, 256, 129), (8, 8, 5)])
def test_parts_of_a_cache(device, fmt, block, D, rows):
    rng = np.random.default_rng(D)
    state = random_cache(rng, 3, 2, rows, D, fmt, block)
    x, values = upload_q8(device, *state, fa.Q8Format(fmt), block), q8.read_back(*state, fmt, block)
    assert np.array_equal(x.dequantize().to_numpy(), values)
    assert np.array_equal(x.narrow(2, 3, rows - 4).narrow(0, 1, 2).narrow(1, 1, 1).dequantize(BF16).to_numpy(),
                          rounded(values[1:3, 1:2, 3:-1], BF16))
    lens = [0, rows - 3, rows + 4]
    out = upload(device, np.full((3, 2, 6, D), 7.0), F16)
    x.dequantize(out=out, row=1, lens=fa.IntTensor(device, lens))
    want = np.full((3, 2, 6, D), 7.0, np.float32)
    for b in range(3):
        for i in range(6):
            place = 1 + lens[b] + i
            if place < rows:
                want[b, :, i] = rounded(values[b, :, place], F16)
    assert np.array_equal(out.to_numpy().astype(np.float32), want)
    assert x.dequantize(rows=0).to_numpy().shape == (3, 2, 0, D)


# ---- the growable cache --------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt, block, D, limit", [(INT8, 1, 64, 50), (E4M3, 8, 72, 50), (INT8, 64, 128, 100), (E4M3, 16, 256, 37), (INT8, 64, 64, 20)])
def test_growing_and_sliding(device, fmt, block, D, limit):
    """Appends up to and far beyond the limit against a cache that keeps every row in place: views, lengths and what they read back."""
    rng = np.random.default_rng(limit + D)
    B, H = 2, 2
    cache = fa.Q8KvCache(2, limit, fa.Q8Format(fmt), block, device)
    wide = fa.KvCache(2, limit, F32, device)
    total = 0
    for n in [1, 3, 1, 5, 20, 1, 1, 2, 9, 1, 1, 30, 1, 1, 1, limit, 1, 4, limit + 3, 1, 2, 1] + [limit // 2 + 1] * 6 + [1] * 7:
        k, v = normals(rng, (B, H, n, D), F16), normals(rng, (B, H, n, D), F16)
        k8, v8 = cache.append(device, upload(device, k, F16), upload(device, v, F16))
        wk, wv = wide.append(device, upload(device, k, F32), upload(device, v, F32))
        total += n
        kept = min(total, limit)
        assert k8.shape == v8.shape == (B, H, kept, D) and cache.current_seq_len() == kept == wide.current_seq_len()
        assert cache.allocated_seq_len() == wide.allocated_seq_len()
        for x8, x in ((k8, wk), (v8, wv)):
            got, want = x8.dequantize().to_numpy(), x.to_numpy()
            # a code is at most half a step off and each of the regrowths of a block's scale adds another half at most; steps: a 127th of the
            # largest element in int8, an eighth of the element's power of two in e4m3
            growths = 1 if block == 1 else 10
            step = 5.0 / 127 if fmt == INT8 else np.maximum(np.abs(want) / 8, 5.0 / 448 / 512)
            assert (np.abs(got - want) <= growths * step / 2 * 1.01).all()
    cache.reset()
    assert cache.current_seq_len() == 0 and cache.allocated_seq_len() == 0
    k = normals(rng, (1, 3, 4, 40), F32)  # another model's shape
    k8, v8 = cache.append(device, upload(device, k, F32), upload(device, k, F32))
    empty = np.zeros((1, 3, 4, 40), np.uint8), np.zeros((1, 3, -(-4 // block)), np.float32)
    assert np.array_equal(k8.dequantize().to_numpy(), q8.read_back(*expected(*empty, k, [0], fmt, block), fmt, block))


def test_cache_steps_with_rotation(device):
    """qkv_rope_append across the limit: the rows that stay are rotated by their own positions."""
    rng = np.random.default_rng(12)
    D, limit = 64, 16
    cache, wide = fa.Q8KvCache(2, limit, device=device), fa.KvCache(2, limit, F32, device)
    rope = fa.RopeCache(D, 100, 10000.0, device)
    norm = fa.RmsNorm(rng.normal(1, 0.3, D).astype(np.float32), None, 1e-6, F32, device)
    pos = 0
    for n in [3, 1, 20, 1, 1, 30, 1]:
        q, k, v = (normals(rng, (1, h, n, D), F16) for h in (4, 2, 2))
        t = [upload(device, x, F16) for x in (q, k, v)]
        got_q, k8, v8 = cache.qkv_rope_append(rope, *t, pos, q_norm=norm, k_norm=norm)
        want_q, wk, wv = wide.qkv_rope_append(rope, *t, pos, q_norm=norm, k_norm=norm)
        assert np.array_equal(got_q.to_numpy(), want_q.to_numpy())
        for x8, x in ((k8, wk), (v8, wv)):
            rows = x.to_numpy()
            s = np.maximum(np.abs(rows).max(-1) * (np.float32(1) / np.float32(127)), q8.LEAST_SCALE)
            assert np.array_equal(x8.dequantize().to_numpy(), q8.read_back(q8.encode(rows, s[..., None], INT8), s, INT8, 1))
        pos += n
    k8, v8 = cache.append_rope(rope, t[1], t[2], pos)
    assert k8.shape == (1, 2, 16, 64)


def test_cache_refusals_leave_it_as_it_was(device):
    rng = np.random.default_rng(13)
    cache = fa.Q8KvCache(2, 16, fa.Q8Format.INT8, 8, device)
    k = upload(device, normals(rng, (1, 2, 5, 64), F16), F16)
    k8, _ = cache.append(device, k, k)
    before = k8.dequantize().to_numpy()
    other = upload(device, normals(rng, (1, 3, 5, 64), F16), F16)
    with pytest.raises(fa.InvalidArgument, match="does not match"):
        cache.append(device, other, other)
    rope = fa.RopeCache(64, 8, 10000.0, device)
    with pytest.raises(fa.InvalidArgument, match="positions"):
        cache.append_rope(rope, k, k, 5)
    a = fa.CQ8AppendArgs()
    a.k_new, a.v_new, a.in_dtype = k._c4(), k._c4(), F16
    a.lens = fa.IntTensor(device, [0]).buffer.ptr
    ka, va = fa.CQ8Tensor(), fa.CQ8Tensor()
    assert fa.lib().fhip_q8_cache_append(cache.handle, device.stream, ctypes.byref(a), ctypes.byref(ka), ctypes.byref(va)) == fa.ERR_INVALID_ARG
    assert cache.current_seq_len() == 5 and np.array_equal(k8.dequantize().to_numpy(), before)


def test_rows_behind_32_bits(device):
    """A row whose bytes lie more than 2^32 into the view."""
    D, rows = 256, (1 << 24) + 1000
    codes = fa.Buffer(device, rows * D)
    scales = fa.Buffer(device, 4 * rows)
    x = fa.Q8Tensor(codes, scales, (1, 1, rows, D), fa.Q8Format.INT8, 1)
    rng = np.random.default_rng(14)
    k = normals(rng, (1, 1, 3, D), F32)
    t = upload(device, k, F32)
    x.append(x, t, t, rows - 3)  # keys and values are the same rows
    s = np.maximum(np.abs(k).max(-1) * (np.float32(1) / np.float32(127)), q8.LEAST_SCALE)
    want = q8.read_back(q8.encode(k, s[..., None], INT8), s, INT8, 1)
    assert np.array_equal(x.dequantize(row=rows - 3).to_numpy(), want)
    assert np.array_equal(x.narrow(2, rows - 2, 2).dequantize().to_numpy(), want[:, :, 1:])


@pytest.mark.parametrize("n", [3, 5000])
@pytest.mark.parametrize("normed", [False, True])
def test_strides_of_64_bits(device, normed, n):
    """Batch strides beyond 31 bits (of a batch of one, which never steps) change nothing."""
    rng = np.random.default_rng(n)
    shape = (1, 8, n, 128)
    tensors = [upload(device, normals(rng, shape, F16), F16) for _ in range(3)]
    far = [fa.Tensor(t.buffer, F16, shape, [1 << 40] + list(t.strides[1:])) for t in tensors]
    norm = fa.RmsNorm(np.linspace(0.5, 1.5, 128, dtype=np.float32), None, 1e-6, F32, device) if normed else None
    rope = fa.RopeCache(128, n, 10000.0, device)
    got = []
    for (q, k, v), wide in ((tensors, False), (far, True)):
        k8, v8 = (fa.Q8Tensor.empty(device, shape, fa.Q8Format(INT8), 1) for _ in range(2))
        if wide:
            k8, v8 = (fa.Q8Tensor(x.codes, x.scales, shape, x.format, 1, (1 << 40,) + x.strides[1:], 0, (1 << 40,) + x.scale_strides[1:]) for x in (k8, v8))
        out = k8.append(v8, k, v, 0, rope=rope, k_norm=norm, q=q, q_norm=norm)
        got.append([out.to_numpy(), k8.dequantize().to_numpy(), v8.dequantize().to_numpy()])
    for near, far_ in zip(*got):
        assert np.array_equal(near, far_)


@pytest.mark.parametrize("B, rows", [(1, (1 << 25) + 41), (5, 1 << 23)])
def test_reading_back_in_parts(device, B, rows):
    """More than 2^30 pieces of eight codes, of one sequence and of five (which share their rows): a launch takes no more."""
    D = 256
    x = fa.Q8Tensor.empty(device, (1, 1, rows, D), fa.Q8Format.INT8, 1)
    rng = np.random.default_rng(3)
    places = [0, min(1 << 25, rows) - 2, rows - 4]
    for at in places:
        t = upload(device, normals(rng, (1, 1, 4, D), F32), F32)
        x.append(x, t, t, min(at, rows - 4))
    whole = fa.Q8Tensor(x.codes, x.scales, (B, 1, rows, D), x.format, 1, (0,) + x.strides[1:], 0, (0,) + x.scale_strides[1:])
    out = whole.dequantize(fa.F16)
    for at in places:
        at = min(at, rows - 4)
        want = x.narrow(2, at, 4).dequantize(fa.F16).to_numpy()
        assert np.abs(want).max() > 0
        for b in range(B):
            part = fa.Tensor(out.buffer, fa.F16, (1, 1, 4, D), (4 * D, 4 * D, D, 1), (b * rows + at) * D)
            assert np.array_equal(part.to_numpy(), want)


@pytest.mark.parametrize("block", [1, 16])
def test_more_rows_than_a_launch_takes(device, block):
    """A call whose rows would need 2^32 lanes and more is refused (all but the first rows would lie outside the cache)."""
    row = upload(device, np.ones((1, 1, 1, 128), np.float32), F32)
    many = fa.Tensor(row.buffer, F32, (1, 1, 1 << 29, 128), (0, 0, 0, 1))
    k8, v8 = (fa.Q8Tensor.empty(device, (1, 1, 16, 128), fa.Q8Format(INT8), block) for _ in range(2))
    with pytest.raises(fa.FhipError, match="lanes"):
        k8.append(v8, many, many, 0, lens=fa.IntTensor(device, [0]))
    assert not k8.dequantize().to_numpy().any()
