"""Forms of the 8-bit attention kernels that only some calls reach: workgroups of eight wavefronts, and mask tensors at every padded head
size, format and block."""
import ctypes

import numpy as np
import pytest

import floneum_amd as fa
from oracle import q8
from q8_helpers import download_q8, random_cache, rounded, upload, upload_q8
from test_q8 import attn
from test_q8_attention_gpu import Call, positions_mask

F32, F16, BF16 = fa.F32, fa.F16, fa.BF16
INT8, E4M3 = q8.INT8, q8.E4M3


def workspace(B, Hkv, D, dtype):
    need = ctypes.c_size_t()
    a = attn(B=B, H=Hkv, Hkv=Hkv, Sq=65, Skv=300, D=D, dtype=dtype)
    assert fa.lib().fhip_q8_attention_workspace_bytes(ctypes.byref(a), 256, ctypes.byref(need)) == fa.OK
    return need.value


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 72, 128])
def test_where_eight_wavefronts_begin(D, dtype):
    """Workgroups of 256 columns that fill the chip, one on each of its 256 CUs, have eight wavefronts and leave the keys whole; one KV head less, and
    those of 128 columns have room for two shares of the keys."""
    assert workspace(8, 32, D, dtype) == 0 and workspace(16, 16, D, dtype) == 0
    assert workspace(1, 255, D, dtype) > 0 and workspace(8, 31, D, dtype) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("D", [40, 64, 72, 128])
@pytest.mark.parametrize("H, Sq, Skv", [(32, 65, 65), (64, 40, 130), (32, 33, 64)])
def test_eight_wavefronts(device, H, Sq, Skv, D, fmt, dtype):
    B, Hkv = 8, 32
    assert B * Hkv >= device.compute_units
    c = Call(device, B, H, Hkv, Sq, Skv, D, dtype, fmt, 1)
    at = Skv - Sq
    c.check(positions_mask(Sq, Skv, [at]), analytic=(True, at, 0))
    c.check(positions_mask(Sq, Skv, [at], 17), analytic=(True, at, 17))
    lens = [Skv, 0, 1, 31, 33, 64, 65, Skv - 1]
    hidden = np.broadcast_to(np.arange(Skv) >= np.asarray(lens)[:, None, None, None], (B, 1, Sq, Skv))
    c.check(hidden, kv_lens=fa.IntTensor(device, lens))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, fmt, D", [(F16, INT8, 128), (BF16, E4M3, 128), (F32, INT8, 128), (F16, E4M3, 64), (F32, E4M3, 64), (BF16, INT8, 72)])
def test_eight_wavefronts_over_several_tiles(device, dtype, fmt, D):
    """Tiles that are staged while others are multiplied, blocks of columns that end inside a wavefront, sequences at positions of their own."""
    B, Hkv, Sq, Skv = 8, 32, 300, 337
    c = Call(device, B, Hkv, Hkv, Sq, Skv, D, dtype, fmt, 1, first=0)
    starts = [37, 0, 5, 36, 20, 1, 30, 12]
    c.check(positions_mask(Sq, Skv, starts), analytic=(True, 0, 0), q_positions=fa.IntTensor(device, starts))
    lens = [s + Sq for s in starts]
    c.check(positions_mask(Sq, Skv, starts, 100, lens), analytic=(True, 0, 100), q_positions=fa.IntTensor(device, starts),
            kv_lens=fa.IntTensor(device, lens))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
def test_eight_wavefronts_in_blocks(device, dtype):
    """Scales of blocks of 16 rows that begin inside one, grouped heads, one sequence of several blocks of columns."""
    Hkv, Sq, Skv = 32, 1100, 90
    c = Call(device, 1, 2 * Hkv, Hkv, Sq, Skv, 64, dtype, INT8, 16, first=5)
    assert Hkv * -(-2 * Sq // 256) >= device.compute_units
    c.check()
    c.check(positions_mask(Sq, Skv, [0]), analytic=(True, 0, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("block, first", [(1, 0), (16, 5)])
@pytest.mark.parametrize("D", [64, 80, 128, 192, 256])
@pytest.mark.parametrize("Sq, Skv", [(2, 100), (40, 100), (33, 65), (70, 300)])
def test_mask_tensors(device, Sq, Skv, D, block, first, fmt, dtype):
    B = 2
    c = Call(device, B, 4, 2, Sq, Skv, D, dtype, fmt, block, first=first)
    low = {F32: -3.4028235e38, F16: -65504.0, BF16: -3.3895314e38}[dtype]
    m = rounded(c.rng.standard_normal((Sq, Skv)).astype(np.float32), dtype)
    m[:, 7], m[-1, 20:] = -np.inf, -np.inf
    m[0, 40:60] = low
    m[1] = -np.inf                              # a row without a key
    hidden = np.broadcast_to(np.isinf(m), (B, 1, Sq, Skv))
    add = np.where(np.isinf(m), 0.0, np.maximum(m.astype(np.float64), -1e4))
    c.check(hidden, add, mask=(upload(device, m, dtype), fa.MaskKind.QKMask))
    c.check(hidden, add, mask=(upload(device, m, dtype, (1, 0)), fa.MaskKind.QKMask))
    pad = np.zeros((B, Skv), np.float32)
    pad[0, :9], pad[1, 50:] = -np.inf, -np.inf  # padded on the left and on the right
    pad[0, 30] = -0.5
    c.check(np.isinf(pad)[:, None, None], np.where(np.isinf(pad), 0.0, pad)[:, None, None], mask=(upload(device, pad, dtype), fa.MaskKind.BatchKeyMask))
    lens = [0, 64]
    hidden = np.isinf(pad)[:, None, None] | (np.arange(Skv) >= np.asarray(lens)[:, None, None, None])
    c.check(hidden, np.where(np.isinf(pad), 0.0, pad)[:, None, None], mask=(upload(device, pad, dtype), fa.MaskKind.BatchKeyMask),
            kv_lens=fa.IntTensor(device, lens))


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", [INT8, E4M3])
@pytest.mark.parametrize("block, n", [(1, 1), (1, 3), (8, 1), (8, 3), (64, 5)])
def test_rows_written_over(device, fmt, block, n):
    """New rows in front of others: those of the same block are lost with its scale, those of later blocks (with blocks of one token, all) stay as they
    were, bit for bit, and so do the blocks in front."""
    rng = np.random.default_rng(block + n)
    B, H, rows, D, at = 2, 2, 200, 64, 66
    state = [random_cache(rng, B, H, rows, D, fmt, block) for _ in range(2)]
    k8, v8 = (upload_q8(device, *s, fa.Q8Format(fmt), block) for s in state)
    new = [rng.standard_normal((B, H, n, D)).astype(np.float32) * np.float32(4) for _ in range(2)]
    k8.append(v8, upload(device, new[0], F32), upload(device, new[1], F32), at)
    end = -(-(at + n) // block)  # the first block behind the new rows
    for t, (codes, scales), x in zip((k8, v8), state, new):
        got, got_scales = download_q8(t)
        want, want_scales = codes.copy(), scales.copy()
        for b in range(B):
            for h in range(H):
                q8.append_rows(want[b, h], want_scales[b, h], x[b, h], at, fmt, block)
        assert np.array_equal(got_scales, want_scales)
        assert np.array_equal(got[:, :, end * block:], codes[:, :, end * block:]) and np.array_equal(got_scales[:, :, end:], scales[:, :, end:])
        assert np.array_equal(got[:, :, :at // block * block], codes[:, :, :at // block * block])
        written = q8.code_values(got[:, :, at:at + n], fmt), q8.code_values(want[:, :, at:at + n], fmt)
        assert np.array_equal(*written)


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("block, n", [(1, 7), (16, 1), (16, 40)])
def test_tables_at_any_f32(device, block, n, interleaved):
    """Rotation tables that begin at any f32, as the wide cache's calls take them: the same bits as tables at the start of their memory."""
    from q8_helpers import _bytes_to
    rng = np.random.default_rng(n)
    B, H, D = 2, 2, 72
    rope = fa.RopeCache(D, 100, 10000.0, device)
    k, v = (upload(device, rng.standard_normal((B, H, n, D)), F32) for _ in range(2))
    q = upload(device, rng.standard_normal((B, 4, n, D)), F32)
    got = []
    for ahead in (0, 1, 3):
        memory = [_bytes_to(device, np.concatenate([np.full(ahead, 9, np.float32), t.ravel(), np.full(4, 9, np.float32)]))
                  for t in (rope.cos_host, rope.sin_host)]
        tables = fa.CRopeTables(*(m.ptr + 4 * ahead for m in memory), 100, 5, int(interleaved))
        k8, v8 = (fa.Q8Tensor.empty(device, (B, H, 60, D), fa.Q8Format.INT8, block) for _ in range(2))
        out = fa.Tensor.empty(device, q.shape, F32)
        a = fa.CQ8AppendArgs()
        a.k, a.v, a.row, a.rope = k8._c(), v8._c(), 3, ctypes.pointer(tables)
        a.k_new, a.v_new, a.in_dtype = k._c4(), v._c4(), F32
        a.q, a.q_out, a.q_dtype, a.q_out_dtype = q._c4(), out._c4(), F32, F32
        fa.check(fa.lib().fhip_q8_append(device.stream, ctypes.byref(a)))
        got.append([out.to_numpy(), *download_q8(k8), *download_q8(v8)])
    for other in got[1:]:
        assert all(np.array_equal(x, y) for x, y in zip(got[0], other))
    assert np.array_equal(got[0][0], q8.rope(q.to_numpy(), rope.cos_host[5:5 + n], rope.sin_host[5:5 + n], interleaved))
