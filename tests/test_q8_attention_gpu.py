"""Attention over the 8-bit cache on the GPU against the same in 64 bits, within the roundings that its description allows."""
import numpy as np
import pytest

import floneum_amd as fa
from oracle import q8
from q8_helpers import attention_bound, random_cache, rounded, spread, upload, upload_q8

pytestmark = pytest.mark.gpu

F32, F16, BF16 = fa.F32, fa.F16, fa.BF16
INT8, E4M3 = q8.INT8, q8.E4M3


class Call:
    """A call's inputs on both sides."""

    def __init__(self, device, B, H, Hkv, Sq, Skv, D, dtype, fmt, block, seed=0, std=1.0, first=0):
        self.rng = np.random.default_rng(seed + 1000 * D + Skv)
        self.device, self.dtype, self.fmt, self.block, self.first = device, dtype, fmt, block, first
        self.scale = D ** -0.5
        self.q = rounded(self.rng.standard_normal((B, H, Sq, D)).astype(np.float32) * np.float32(std), dtype)
        self.k_state, self.v_state = (random_cache(self.rng, B, Hkv, Skv, D, fmt, block, first=first) for _ in range(2))

    def values(self):
        return [q8.read_back(*s, self.fmt, self.block, self.first).astype(np.float64) for s in (self.k_state, self.v_state)]

    def v_scales(self):
        return self.v_state[1][..., (self.first + np.arange(self.v_state[0].shape[2])) // self.block].astype(np.float64)

    def tensors(self):
        return [upload_q8(self.device, *s, fa.Q8Format(self.fmt), self.block, self.first) for s in (self.k_state, self.v_state)]

    def check(self, hidden=None, add=None, out_dtype=None, tensors=None, got=None, **kw):
        if got is None:
            got = upload(self.device, self.q, self.dtype).flash_attention(*(tensors or self.tensors()), self.scale, out_dtype=out_dtype, **kw).to_numpy()
        got = np.asarray(got, np.float64)
        k, v = self.values()
        lost = [np.isnan(x).any(-1) for x in (k, v)]  # rows with a scale that is NaN, which nobody may see here
        k, v = (np.where(bad[..., None], 0.0, x) for bad, x in zip(lost, (k, v)))
        q = self.q.astype(np.float64)
        want, mass, top, p = q8.attention(q, k, v, self.scale, hidden, add)
        out_dtype = self.dtype if out_dtype is None else out_dtype
        v_scales = self.v_scales()
        bound = attention_bound(np.nan_to_num(want), np.nan_to_num(mass), top, p, q, k, self.scale, v_scales, self.fmt, self.dtype, out_dtype)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        off = np.abs(np.nan_to_num(got) - np.nan_to_num(want))
        assert (off <= bound).all(), (float((off / bound).max()), np.argwhere(off > bound)[:4], float(off.max()))


def positions_mask(Sq, Skv, offsets, window=0, lens=None):
    """hidden [B,1,Sq,Skv] of a causal mask with query row 0 of sequence b at offsets[b]."""
    at = np.asarray(offsets)[:, None, None, None] + np.arange(Sq)[:, None]
    key = np.arange(Skv)
    hidden = key > at
    if window:
        hidden = hidden | (key + window <= at)
    if lens is not None:
        hidden = hidden | (key >= np.asarray(lens)[:, None, None, None])
    return hidden


# ---- shapes and types -----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [8, 40, 64, 72, 80, 96, 128, 136, 192, 200, 256])
def test_head_dims(device, D, dtype, fmt):
    Call(device, 2, 4, 2, 1, 133, D, dtype, fmt, 1).check()


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("Skv", [1, 2, 15, 16, 31, 32, 33, 63, 127, 128, 129, 255, 257, 1000, 4099])
def test_lengths(device, Skv, dtype):
    Call(device, 1, 8, 2, 1, Skv, 64, dtype, INT8, 1).check()


@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("block", [1, 8, 16, 32, 64])
@pytest.mark.parametrize("Skv, first", [(5, 0), (97, 5), (700, 7)])
def test_blocks(device, Skv, first, block, fmt):
    first = first if block > 1 else 0
    Call(device, 2, 4, 4, 1, Skv, 128, BF16, fmt, block, first=first).check()
    Call(device, 1, 4, 1, 3, Skv, 64, F32, fmt, block, first=first).check()


@pytest.mark.parametrize("H, Hkv", [(1, 1), (7, 7), (8, 1), (12, 4), (32, 2), (48, 1), (6, 2)])
def test_head_groups(device, H, Hkv):
    Call(device, 2, H, Hkv, 1, 300, 64, F16, INT8, 1).check()
    Call(device, 1, H, Hkv, 5, 300, 128, BF16, E4M3, 8).check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("Sq, Skv, D", [(2, 130, 64), (4, 4001, 256), (7, 90, 128), (16, 16, 64), (17, 200, 96), (33, 33, 128), (64, 500, 64),
                                        (100, 100, 80), (129, 1003, 128), (200, 333, 192), (300, 300, 256), (257, 640, 72)])
def test_query_rows_under_a_causal_mask(device, Sq, Skv, D, dtype):
    fmt, block = (INT8, 1) if Skv % 2 else (E4M3, 16)
    c = Call(device, 1, 4, 2, Sq, Skv, D, dtype, fmt, block)
    hidden = positions_mask(Sq, Skv, [Skv - Sq])
    c.check(hidden, analytic=(True, Skv - Sq, 0))
    c.check()
    c.check(positions_mask(Sq, Skv, [Skv - Sq], 40), analytic=(True, Skv - Sq, 40))
    c.check(out_dtype=F32)


def test_batches(device):
    Call(device, 33, 4, 2, 1, 77, 64, F16, INT8, 1).check()
    Call(device, 5, 32, 8, 1, 600, 128, F16, INT8, 1).check()


@pytest.mark.parametrize("dtype", [F32, F16])
def test_long_rows(device, dtype):
    Call(device, 1, 8, 2, 1, 40000, 64, dtype, INT8, 1, std=2.0).check()
    Call(device, 1, 4, 2, 6, 20011, 128, dtype, E4M3, 32).check(positions_mask(6, 20011, [20005]), analytic=(True, 20005, 0))


@pytest.mark.parametrize("fmt", [INT8, E4M3])
def test_f32_precision(device, fmt):
    """Each probability is off by a few 2^-24 of itself and by itself (two terms of 11 bits and the rounding of the score), so the output is off
    by as much, relative to its own size although it is a small difference of large sums: below 2^-20 in the mean.  One key whose two terms do not
    belong together (off by 2^-12) shows."""
    for seed in range(4):
        c = Call(device, 1, 8, 1, 1, 4096, 128, F32, fmt, 1, seed=seed)
        got = upload(device, c.q, F32).flash_attention(*c.tensors(), c.scale).to_numpy().astype(np.float64)
        k, v = (q8.code_values(s[0], fmt) * s[1][..., None].astype(np.float64) for s in (c.k_state, c.v_state))
        want = q8.attention(c.q, k, v, float(np.float32(c.scale)))[0]
        off = np.linalg.norm(got - want, axis=-1) / np.linalg.norm(want, axis=-1)
        assert off.max() < 2.0 ** -20, off


# ---- masks ------------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("Sq", [1, 3, 70])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lengths_of_their_own(device, Sq, dtype):
    """Sequences of no key, one key, all keys and beyond; what lies behind their last row is not seen, whatever it is."""
    lens = [0, 1, 31, 32, 200, 1000, -5]
    B, Skv = len(lens), 200
    c = Call(device, B, 4, 2, Sq, Skv, 64, dtype, E4M3, 1)
    for b, n in enumerate(lens):
        n = max(n, 0)
        for codes, scales in (c.k_state, c.v_state):
            codes[b, :, n:], scales[b, :, n:] = 0x7F, np.nan  # 8-bit NaN and scales that are NaN
    hidden = np.broadcast_to(np.arange(Skv) >= np.asarray(lens)[:, None, None, None], (B, 1, Sq, Skv))
    c.check(hidden, kv_lens=fa.IntTensor(device, lens))


@pytest.mark.parametrize("window", [0, 1, 50])
@pytest.mark.parametrize("Sq, block", [(1, 1), (4, 8), (50, 64), (130, 1)])
def test_positions_of_their_own(device, Sq, block, window):
    """q_positions with kv_lens: a batch whose sequences end at different places, and rows without a key."""
    lens = [Sq, Sq + 1, 199, 300, Sq + 70]
    starts = [n - Sq for n in lens]
    starts[3] = 2000  # beyond the cache: under a window nothing is left to see
    c = Call(device, len(lens), 4, 2, Sq, 300, 64, F16, INT8, block)
    hidden = positions_mask(Sq, 300, [3 + s for s in starts], window, lens)
    c.check(hidden, kv_lens=fa.IntTensor(device, lens), analytic=(True, 3, window), q_positions=fa.IntTensor(device, starts))


def test_rows_hidden_by_position_may_hold_anything(device):
    """Keys that some rows see and others do not, with scales that are NaN, are nothing to those that do not."""
    c = Call(device, 1, 4, 2, 4, 100, 64, F16, INT8, 1)
    for state in (c.k_state, c.v_state):
        state[1][:, :, 99] = np.nan
    hidden = positions_mask(4, 100, [96])
    q = upload(device, c.q, F16)
    got = q.flash_attention(*c.tensors(), c.scale, analytic=(True, 96, 0)).to_numpy().astype(np.float64)
    assert np.isnan(got[:, :, 3]).all()
    hidden[:, :, 3] = True
    c.check(hidden, got=got)


@pytest.mark.parametrize("which", [0, 1])
def test_visible_rows_that_are_nan(device, which):
    c = Call(device, 1, 2, 2, 1, 100, 64, F16, E4M3, 8)
    (c.k_state, c.v_state)[which][1][0, 1, 4] = np.nan
    got = upload(device, c.q, F16).flash_attention(*c.tensors(), c.scale).to_numpy()
    assert np.isnan(got[0, 1]).all() and not np.isnan(got[0, 0]).any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("Sq", [1, 5, 40, 150])
def test_mask_tensors(device, Sq, dtype):
    B, Skv = 2, 260
    c = Call(device, B, 4, 2, Sq, Skv, 64, dtype, INT8, 1)
    low = {F32: -3.4028235e38, F16: -65504.0, BF16: -3.3895314e38}[dtype]
    m = rounded(c.rng.standard_normal((Sq, Skv)).astype(np.float32), dtype)
    m[:, 7] = -np.inf
    m[0, 20:90] = low
    if Sq > 1:
        m[1] = -np.inf          # a row without a key
    if Sq > 4:
        m[4] = low              # a row whose keys are all equally far down
    t = upload(device, m, dtype)
    add = np.where(np.isinf(m), 0.0, m.astype(np.float64))
    row_low = (m == low).all(-1)
    if dtype != F16 and Sq > 4:  # scores vanish beside such a value: all keys weigh the same
        mean = np.repeat(c.values()[1].mean(2, keepdims=True), 2, 1)
        got = upload(device, c.q, dtype).flash_attention(*c.tensors(), c.scale, (t, fa.MaskKind.QKMask)).to_numpy()
        assert np.abs(got[:, :, row_low] - mean).max() < 2.0 ** -7
    add[row_low] = 0.0 if dtype != F16 else add[row_low]
    hidden = np.isinf(m)[None, None]
    if dtype == F16 and Sq > 4:  # sums of about 65504 keep 2^-8 of the scores
        add[4], m[4] = 0.0, 0.0
        t = upload(device, m, dtype)
    elif Sq > 4:
        m[4], add[4] = 0.0, 0.0
        t = upload(device, m, dtype)
    add[0, 20:90] = -1e4
    hidden = np.broadcast_to(hidden | False, (B, 4, Sq, Skv))
    c.check(hidden, add, mask=(t, fa.MaskKind.QKMask))
    pad = np.zeros((B, Skv), np.float32)
    pad[0, 100:], pad[1, 3] = -10000.0, -np.inf
    c.check(np.broadcast_to(np.isinf(pad)[:, None, None], (B, 4, Sq, Skv)), np.where(np.isinf(pad), 0, pad)[:, None, None],
            mask=(upload(device, pad, dtype), fa.MaskKind.BatchKeyMask))
    # a transposed mask
    c.check(hidden, add, mask=(upload(device, m, dtype, (1, 0)), fa.MaskKind.QKMask))


def test_no_keys(device):
    c = Call(device, 2, 4, 2, 3, 10, 64, F16, INT8, 1)
    k, v = (t.narrow(2, 4, 0) for t in c.tensors())
    out = upload(device, c.q, F16).flash_attention(k, v, c.scale)
    assert (out.to_numpy() == 0).all()
    assert upload(device, c.q, F16).narrow(2, 0, 0).flash_attention(*c.tensors(), c.scale).shape == (2, 4, 0, 64)


# ---- values -----------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scales_far_apart(device, dtype):
    """Values of almost nothing on the keys that count (a first token that attention rests on), large ones on the others; queries and keys
    whose products need the scales' whole range."""
    c = Call(device, 1, 4, 2, 2, 150, 64, dtype, INT8, 1)
    c.v_state[1][:, :, ::2] *= np.float32(2.0 ** -40)
    c.v_state[1][:, :, 5] *= np.float32(2.0 ** 30)
    c.k_state[1][:, :, :] *= np.float32(2.0 ** 60 if dtype == F32 else 2.0 ** 8)
    c.q = rounded(c.q * np.float32(2.0 ** -60 if dtype == F32 else 2.0 ** -8), dtype)
    c.check(out_dtype=F32)
    c.v_state[1][:, :, 6] = 0.0
    c.v_state[0][:, :, 6] = 0
    c.check(out_dtype=F32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D, Sq, Skv", [(64, 40, 700), (128, 300, 449), (256, 33, 1500), (192, 65, 64), (128, 64, 65)])
def test_rising_maximum(device, dtype, D, Sq, Skv):
    """Scores that grow along the keys, slowly enough that a row's maximum moves a little in every tile; then values' scales that grow."""
    c = Call(device, 1, 4, 2, Sq, Skv, D, dtype, INT8, 1)
    c.k_state[1][:] *= np.linspace(0.25, 8.0, Skv, dtype=np.float32)
    c.check(out_dtype=F32)
    c.v_state[1][:] *= np.exp2(np.linspace(-3.0, 3.0, Skv, dtype=np.float32))
    offset = max(0, Skv - Sq)
    c.check(hidden=positions_mask(Sq, Skv, [offset]), analytic=(True, offset, 0), out_dtype=F32)


def test_queries_of_any_size(device):
    for power in (-140, -100, 0, 60):
        c = Call(device, 1, 2, 2, 2, 64, 64, F32, INT8, 1)
        c.q = (c.q * np.float32(2.0) ** min(power, 0) * np.float32(2.0) ** max(power, 0)).astype(np.float32)
        c.scale = 2.0 ** -(max(power, 0) + 3)
        c.check()
    c = Call(device, 1, 2, 2, 1, 64, 64, F32, INT8, 1)
    c.q[:] = 0.0
    c.check()


def test_infinite_queries(device):
    c = Call(device, 1, 2, 2, 1, 64, 64, F16, INT8, 1)
    c.q[0, 0, 0, 3] = np.inf
    c.q[0, 1, 0, 3] = np.nan
    assert np.isnan(upload(device, c.q, F16).flash_attention(*c.tensors(), c.scale).to_numpy()).all()


# ---- layouts, streams, graphs -------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("Sq", [1, 37])
def test_layouts(device, Sq):
    """Queries with gaps, an output as the projection behind attention reads it, one cache shared by the batch and by heads."""
    B, H, Hkv, Skv, D = 3, 4, 2, 90, 72
    c = Call(device, 1, H, Hkv, Sq, Skv, D, F16, INT8, 16)
    q = rounded(c.rng.standard_normal((B, H, Sq, D)).astype(np.float32), F16)
    whole = np.zeros((B, Sq, H, 2 * D), np.float32)
    whole[..., ::2] = q.transpose(0, 2, 1, 3)
    base = upload(device, whole, F16)
    tq = fa.Tensor(base.buffer, F16, (B, H, Sq, D), (base.strides[0], base.strides[2], base.strides[1], 2))
    memory, out = spread(device, (B, Sq, H, D), F16, (1, 2, 1, 3), 9.0)
    k, v = c.tensors()
    k, v = (fa.Q8Tensor(t.codes, t.scales, (B, Hkv, Skv, D), t.format, t.block_tokens, (0, *t.strides[1:]), 0, (0, t.scale_strides[1])) for t in (k, v))
    tq.flash_attention(k, v, c.scale, out=out.transpose(1, 2))
    host = memory.to_numpy()
    c.q = q
    c.k_state, c.v_state = (tuple(np.repeat(x, B, 0) for x in s) for s in (c.k_state, c.v_state))
    c.check(got=host[:, ::2, :, ::3].transpose(0, 2, 1, 3))
    host[:, ::2, :, ::3] = 9.0
    assert (host == 9.0).all()


def test_rows_apart(device):
    """A cache whose rows of all heads lie together: [batch, rows, heads, head_dim] seen as [batch, heads, rows, head_dim]."""
    B, Hkv, Skv, D = 2, 3, 150, 64
    c = Call(device, B, 6, Hkv, 1, Skv, D, BF16, E4M3, 1)
    k, v = (upload_q8(device, np.ascontiguousarray(codes.transpose(0, 2, 1, 3)), scales, fa.Q8Format.E4M3, 1) for codes, scales in (c.k_state, c.v_state))
    k, v = (fa.Q8Tensor(t.codes, t.scales, (B, Hkv, Skv, D), t.format, 1, (Skv * Hkv * D, D, Hkv * D), 0, (Hkv * Skv, Skv)) for t in (k, v))
    c.check(tensors=(k, v))


def test_rows_behind_32_bits(device):
    D, rows = 256, (1 << 24) + 1000
    codes, scales = fa.Buffer(device, rows * D), fa.Buffer(device, 4 * rows)
    k8 = fa.Q8Tensor(codes, scales, (1, 1, rows, D), fa.Q8Format.INT8, 1)
    c = Call(device, 1, 2, 1, 1, 300, D, F16, INT8, 1)
    x = q8.read_back(*c.k_state, INT8, 1)
    k8.append(k8, upload(device, x, F32), upload(device, x, F32), rows - 300)
    c.v_state = c.k_state
    got = upload(device, c.q, F16).flash_attention(k8, k8, c.scale, analytic=(True, rows - 1, 300)).to_numpy()
    c.check(got=got)
    c.check(got=upload(device, c.q, F16).flash_attention(k8.narrow(2, rows - 300, 300), k8.narrow(2, rows - 300, 300), c.scale).to_numpy())


def test_two_streams(device):
    """The same calls on two streams of one device at once, each with its own workspace."""
    other = device.with_new_stream()
    calls = [Call(dev, 1, 8, 2, 1, 3000, 128, F16, INT8, 1, seed=s) for s, dev in enumerate((device, other))]
    inputs = [(upload(c.device, c.q, F16), c.tensors()) for c in calls]
    outs = [[], []]
    for _ in range(5):
        for i, (q, kv) in enumerate(inputs):
            outs[i].append(q.flash_attention(*kv, calls[i].scale))
    for c, got in zip(calls, outs):
        first = got[0].to_numpy()
        assert all(np.array_equal(first, x.to_numpy()) for x in got)
        c.check(got=first)


def test_repeatable(device):
    for Sq in (1, 130):
        c = Call(device, 2, 8, 2, Sq, 2500, 128, F32, E4M3, 16)
        q, kv = upload(device, c.q, F32), c.tensors()
        runs = [q.flash_attention(*kv, c.scale).to_numpy() for _ in range(4)]
        assert all(np.array_equal(runs[0], x) for x in runs)


@pytest.mark.parametrize("fmt, block", [(INT8, 1), (E4M3, 16)])
def test_a_captured_step(device, fmt, block):
    """A decode step recorded once and replayed with new rows, lengths and positions on the device: rotation, 8-bit append, attention."""
    import ctypes
    B, H, Hkv, D, rows = 3, 8, 2, 64, 200
    rng = np.random.default_rng(20)
    rope = fa.RopeCache(D, 256, 10000.0, device)
    state = [random_cache(rng, B, Hkv, rows, D, fmt, block) for _ in range(2)]
    k8, v8 = (upload_q8(device, *s, fa.Q8Format(fmt), block) for s in state)
    tq, tk, tv = (upload(device, np.zeros((B, h, 1, D)), F16) for h in (H, Hkv, Hkv))
    lens, after = fa.IntTensor(device, [1] * B), fa.IntTensor(device, [2] * B)
    out = upload(device, np.zeros((B, H, 1, D)), F16)

    def write(t, host):
        host = np.ascontiguousarray(host)
        fa.check(fa.lib().fhip_memcpy_h2d(device.stream, ctypes.c_void_p(t.buffer.ptr), host.ctypes.data_as(ctypes.c_void_p), host.nbytes))

    def step():
        q = k8.append(v8, tk, tv, lens=lens, rope=rope, q=tq)
        q.flash_attention(k8, v8, D ** -0.5, kv_lens=after, analytic=(True, 0, 64), q_positions=lens, out=out)

    step()
    device.synchronize()
    with device.capture() as cap:
        step()
    for turn in range(4):
        at = [int(x) for x in rng.integers(1, rows - 1, B)]
        new = [rounded(rng.standard_normal((B, h, 1, D)).astype(np.float32), F16) for h in (H, Hkv, Hkv)]
        for t, x in zip((tq, tk, tv), new):
            write(t, x.astype(np.float16))
        write(lens, np.asarray(at, np.int32))
        write(after, np.asarray(at, np.int32) + 1)
        before = [x.dequantize(F32).to_numpy() for x in (k8, v8)]
        device.synchronize()
        cap.graph.launch()
        got = out.to_numpy()
        after_rows = [x.dequantize(F32).to_numpy() for x in (k8, v8)]
        cos, sin = (t[at][:, None, None] for t in (rope.cos_host, rope.sin_host))
        c = Call.__new__(Call)
        c.device, c.dtype, c.fmt, c.block, c.first, c.scale, c.rng = device, F16, fmt, block, 0, D ** -0.5, rng
        c.q = rounded(q8.rope(new[0], cos, sin), F16)
        c.values = lambda: [x.astype(np.float64) for x in after_rows]
        c.v_scales = lambda: np.abs(after_rows[1]).max(-1).astype(np.float64)  # (a code of 1 at least)
        hidden = positions_mask(1, rows, at, 64)
        c.check(hidden, got=got)
        for b in range(B):  # nothing but the new rows' blocks has changed
            lo, hi = at[b] // block * block, at[b] // block * block + block
            for x, y in zip(before, after_rows):
                assert np.array_equal(x[b, :, :lo], y[b, :, :lo]) and np.array_equal(x[b, :, hi:], y[b, :, hi:])


def test_a_layer(device):
    """A prompt, single tokens and a draft through the growable cache and attention, beside the same layer on the wide f32 cache: the two
    differ by what 8 bits leave out."""
    rng = np.random.default_rng(21)
    H, Hkv, D = 8, 2, 128
    rope = fa.RopeCache(D, 600, 10000.0, device)
    norm = fa.RmsNorm(rng.normal(1, 0.2, D).astype(np.float32), None, 1e-6, F32, device)
    for fmt, block in ((fa.Q8Format.INT8, 1), (fa.Q8Format.E4M3, 32)):
        cache, wide = fa.Q8KvCache(2, 512, fmt, block, device), fa.KvCache(2, 512, F32, device)
        at = 0
        for n in (200, 1, 1, 1, 5, 1, 130, 1):
            t = [upload(device, rng.standard_normal((1, h, n, D)), F32) for h in (H, Hkv, Hkv)]
            q, k8, v8 = cache.qkv_rope_append(rope, *t, at, q_norm=norm, k_norm=norm)
            wq, k, v = wide.qkv_rope_append(rope, *t, at, q_norm=norm, k_norm=norm)
            at += n
            got = q.flash_attention(k8, v8, D ** -0.5, analytic=(True, at - n, 0)).to_numpy()
            want = wq.flash_attention(k, v, D ** -0.5, analytic=(True, at - n, 0)).to_numpy()
            # values are off by up to half a step, 1/127 of a row's largest (about 4) or 1/16 of a value; scores by a few per cent, too
            assert np.linalg.norm(got - want) < 0.06 * np.linalg.norm(want)
            # and next to attention over what the cache reads back as
            kd, vd = k8.dequantize(F32), v8.dequantize(F32)
            same = q.flash_attention(kd, vd, D ** -0.5, analytic=(True, at - n, 0)).to_numpy()
            assert np.linalg.norm(got - same) < 2e-5 * np.linalg.norm(same)


# ---- refusals -----------------------------------------------------------------------------------------------------------------------------------

def test_refusals(device):
    c = Call(device, 1, 2, 2, 1, 20, 64, F16, INT8, 1)
    q, (k, v) = upload(device, c.q, F16), c.tensors()
    wide = upload(device, np.zeros((1, 2, 20, 64)), F16)
    for bad in (lambda: q.flash_attention(k, wide, 1.0), lambda: q.flash_attention(wide, v, 1.0),
                lambda: q.flash_attention(wide, wide, 1.0, q_positions=fa.IntTensor(device, [0])),
                lambda: q.flash_attention(k, v, 1.0, force_kernel=fa.KERNEL_GENERIC),
                lambda: q.flash_attention(k, v, 1.0, q_positions=fa.IntTensor(device, [0])),
                lambda: q.flash_attention(k, v, 1.0, kv_lens=fa.IntTensor(device, [0, 1])),
                lambda: q.flash_attention(k, v.narrow(2, 0, 19), 1.0),
                lambda: q.flash_attention(k, v, 1.0, out=upload(device, c.q, F16), out_dtype=F32),
                lambda: q.flash_attention(k, v, 1.0, (upload(device, np.zeros((1, 20)), F32), fa.MaskKind.QKMask)),
                lambda: k.append(v, wide, upload(device, np.zeros((1, 2, 20, 64)), F32)),
                lambda: k.append(v, wide, wide, 1),
                lambda: k.append(v, wide, wide, q_out=wide),
                lambda: k.dequantize(row=1, rows=20)):
        with pytest.raises(fa.InvalidArgument):
            bad()
    with pytest.raises(AssertionError):
        q.flash_attention(k, upload_q8(device.with_new_stream(), *c.v_state, fa.Q8Format.INT8, 1), 1.0)


def test_too_little_workspace(device):
    import ctypes
    c = Call(device, 1, 2, 2, 1, 2000, 64, F16, INT8, 1)
    q, (k, v) = upload(device, c.q, F16), c.tensors()
    out = upload(device, c.q, F16)
    a = fa.CQ8AttnArgs()
    a.q, a.out, a.k, a.v, a.dtype, a.out_dtype, a.scale = q._c4(), out._c4(), k._c(), v._c(), F16, F16, c.scale
    need = ctypes.c_size_t()
    fa.check(fa.lib().fhip_q8_attention_workspace_bytes(ctypes.byref(a), device.compute_units, ctypes.byref(need)))
    assert need.value > 0
    memory = fa.Buffer(device, need.value + 16)
    for ptr, size in ((None, 0), (memory.ptr, need.value - 1), (memory.ptr + 4, need.value)):
        a.workspace, a.workspace_bytes = ptr, size
        assert fa.lib().fhip_q8_attention(device.stream, ctypes.byref(a)) == fa.ERR_WORKSPACE
    a.workspace, a.workspace_bytes = memory.ptr, need.value
    assert fa.lib().fhip_q8_attention(device.stream, ctypes.byref(a)) == fa.OK
    c.check(got=out.to_numpy())


@pytest.mark.parametrize("with_native", [True, False])
def test_both_ways_to_the_library(device, monkeypatch, with_native):
    """The mirror's calls through its native half and through ctypes."""
    assert fa._native is not None
    if not with_native:
        monkeypatch.setattr(fa, "_native", None)
    rng = np.random.default_rng(30)
    rope = fa.RopeCache(64, 64, 10000.0, device)
    norm = fa.RmsNorm(rng.normal(1, 0.2, 64).astype(np.float32), None, 1e-6, F32, device)
    cache = fa.Q8KvCache(2, 64, fa.Q8Format.INT8, 8, device)
    q, k, v = (rng.standard_normal((2, h, 9, 64)).astype(np.float32) for h in (4, 2, 2))
    t = [upload(device, x, F32) for x in (q, k, v)]
    turned, k8, v8 = cache.qkv_rope_append(rope, *t, 3, q_norm=norm, k_norm=norm)
    mask = (upload(device, np.zeros((9, 9)), F32), fa.MaskKind.QKMask)
    got = [turned.flash_attention(k8, v8, 0.125, m, analytic=a, kv_lens=n, q_positions=x) for m, a, n, x in
           ((None, None, None, None), (mask, None, None, None), (None, (True, 0, 4), fa.IntTensor(device, [9, 5]), fa.IntTensor(device, [0, 1])))]
    own = fa.Q8Tensor.empty(device, (2, 2, 20, 64), fa.Q8Format.INT8, 8)
    own2 = fa.Q8Tensor.empty(device, (2, 2, 20, 64), fa.Q8Format.INT8, 8)
    turned2 = own.append(own2, t[1], t[2], 1, lens=fa.IntTensor(device, [2, 2]), counts=fa.IntTensor(device, [9, 9]), rope=rope, start_pos=1, k_norm=norm,
                         q=t[0], q_norm=norm)
    assert np.array_equal(turned.to_numpy(), turned2.to_numpy())
    back = own.narrow(2, 3, 9).dequantize(F32), own2.dequantize(F32, row=1, rows=9, lens=fa.IntTensor(device, [2, 2]))
    for a, b in zip(back, (k8, v8)):
        # (blocks lie elsewhere: 8-bit codes of other scales)
        assert np.abs(a.to_numpy() - b.dequantize(F32).to_numpy()).max() < 5.0 / 127
    want = [turned.flash_attention(k8.dequantize(F32), v8.dequantize(F32), 0.125, m, analytic=a, kv_lens=n) for m, a, n in
            ((None, None, None), (mask, None, None))]
    for a, b in zip(got, want):
        assert np.abs(a.to_numpy() - b.to_numpy()).max() < 1e-5
    windowed = got[2].to_numpy()  # row r of sequence 1 sees keys r - 2 .. r + 1 below 5
    assert np.isnan(windowed[1, :, 7:]).all() and np.isfinite(windowed[1, :, :7]).all() and np.isfinite(windowed[0]).all()
    assert not np.array_equal(windowed[0], got[0].to_numpy()[0])


def test_shares_in_any_workspace(device):
    """A workspace that starts with anything, calls of different shapes that follow each other in it, and a recorded call replayed."""
    import ctypes
    for D, Skv, Sq, B in ((64, 3000, 1, 2), (128, 1500, 3, 1), (256, 2000, 1, 3), (192, 9000, 1, 1)):
        c = Call(device, B, 8, 2, Sq, Skv, D, F16, INT8, 1)
        q, kv = upload(device, c.q, F16), c.tensors()
        ws, size = device.workspace(1 << 24)
        for fill in (0, 0xFF, 0x55):
            fa.check(fa.lib().fhip_memset(device.stream, ctypes.c_void_p(ws), fill, size))
            c.check(got=q.flash_attention(*kv, c.scale).to_numpy())
        out = upload(device, c.q, F16)
        with device.capture() as cap:
            q.flash_attention(*kv, c.scale, out=out)
        first = q.flash_attention(*kv, c.scale).to_numpy()
        for _ in range(4):
            fa.check(fa.lib().fhip_memset(device.stream, ctypes.c_void_p(out.buffer.ptr), 0, out.buffer.nbytes))
            cap.graph.launch()
            assert np.array_equal(out.to_numpy(), first)
            q.flash_attention(*kv, c.scale)
        del cap
