"""Attention over the 8-bit cache where numbers are near the ends of f32's range, on both kernels (few rows and many), against the same in
64 bits."""
import numpy as np
import pytest

import floneum_amd as fa
from oracle import q8
from q8_helpers import rounded, upload, upload_q8
from test_q8_attention_gpu import Call, positions_mask

pytestmark = pytest.mark.gpu

F32, F16, BF16 = fa.F32, fa.F16, fa.BF16
INT8, E4M3 = q8.INT8, q8.E4M3


def times_power(x, power):
    """x * 2^power in f32 (in two steps: the power alone may have no f32)."""
    half = power // 2
    return (x * np.float32(2.0 ** half) * np.float32(2.0 ** (power - half))).astype(np.float32)


# ---- scores -------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("power, scale", [(-140, None), (-145, 2.0 ** -20), (0, 1e-44), (-100, 2.0 ** -60), (-30, 2.0 ** -126)])
@pytest.mark.parametrize("D, Sq, Skv", [(64, 40, 65), (128, 130, 130), (256, 40, 200), (64, 2, 65)])
def test_queries_of_almost_nothing(device, dtype, power, scale, D, Sq, Skv):
    """Queries, or a factor of the scores, that leave scores of nothing: every key that a row sees weighs the same, hidden ones nothing."""
    c = Call(device, 1, 4, 2, Sq, Skv, D, dtype, INT8, 1)
    c.q = rounded(times_power(c.q, max(power, -131) if dtype == BF16 else power), dtype)  # (bf16 ends at 2^-133)
    c.scale = c.scale if scale is None else scale
    c.check()
    at = Skv - Sq
    c.check(positions_mask(Sq, Skv, [at]), analytic=(True, at, 0))
    c.check(positions_mask(Sq, Skv, [at], 20), analytic=(True, at, 20))
    c.check(np.broadcast_to(np.arange(Skv) >= 50, (1, 1, Sq, Skv)), kv_lens=fa.IntTensor(device, [50]))
    m = np.where(positions_mask(Sq, Skv, [at])[0, 0], -np.inf, 0.0).astype(np.float32)
    c.check(positions_mask(Sq, Skv, [at]), mask=(upload(device, m, dtype), fa.MaskKind.QKMask))


@pytest.mark.parametrize("Sq, Skv", [(2, 300), (40, 65), (130, 200)])
def test_the_largest_factor(device, Sq, Skv):
    """A factor of the scores whose product with log2 e is beyond f32, with keys and queries whose products are that small."""
    c = Call(device, 1, 4, 2, Sq, Skv, 64, F32, INT8, 1)
    c.q = times_power(c.q, -60)
    c.k_state[1][:] = times_power(c.k_state[1], -70)
    c.scale = 3.2e38
    c.check()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("Sq, Skv", [(2, 300), (40, 65), (130, 200)])
def test_large_factors_of_the_least_products(device, dtype, Sq, Skv):
    """Scores of ordinary size from the least queries of f16, keys of the least scale and a factor of 2^120."""
    c = Call(device, 1, 4, 2, Sq, Skv, 64, dtype, INT8, 1)
    c.q = np.sign(c.q).astype(np.float32) * np.float32(2.0 ** -24)
    c.k_state = np.sign(c.k_state[0].view(np.int8)).astype(np.int8).view(np.uint8), np.full_like(c.k_state[1], q8.LEAST_SCALE)
    c.scale = 2.0 ** 120
    c.check()
    at = Skv - Sq
    c.check(positions_mask(Sq, Skv, [at]), analytic=(True, at, 0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("Sq, Skv", [(2, 300), (40, 65), (130, 200)])
def test_the_least_factors_of_large_products(device, dtype, Sq, Skv):
    """Scores of ordinary size from large queries of f16, keys of 2^123 and a factor that is no normal f32."""
    c = Call(device, 1, 4, 2, Sq, Skv, 64, dtype, INT8, 1)
    c.q = rounded(c.q * np.float32(2.0 ** 12), dtype)
    c.k_state[1][:] = times_power(c.k_state[1], 123)
    c.scale = float(np.float32(1.37 * 2.0 ** -139))
    c.check()
    at = Skv - Sq
    c.check(positions_mask(Sq, Skv, [at]), analytic=(True, at, 0))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("fmt, block", [(INT8, 1), (E4M3, 16)])
@pytest.mark.parametrize("D, Sq, Skv", [(64, 2, 300), (128, 1, 64), (64, 40, 65), (128, 130, 300), (256, 40, 90)])
@pytest.mark.parametrize("power", [-90, 90, 112, 125])
def test_keys_and_queries_far_apart(device, dtype, fmt, block, D, Sq, Skv, power):
    """Scores of ordinary size from keys that are 2^power times the ordinary and queries that are as much smaller."""
    c = Call(device, 1, 4, 2, Sq, Skv, D, dtype, fmt, block)
    c.q = rounded(times_power(c.q, -power), dtype)
    c.k_state[1][:] = times_power(c.k_state[1], power)
    c.check(out_dtype=F32)
    at = Skv - Sq
    c.check(positions_mask(Sq, Skv, [at]), analytic=(True, at, 0), out_dtype=F32)
    m = np.where(positions_mask(Sq, Skv, [at])[0, 0], -np.inf, 0.0).astype(np.float32)
    c.check(positions_mask(Sq, Skv, [at]), mask=(upload(device, m, dtype), fa.MaskKind.QKMask), out_dtype=F32)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("Sq", [2, 40])
def test_keys_of_every_size_at_once(device, dtype, Sq):
    """Keys of 2^110 in front of, beside and behind ordinary ones, which the queries are small enough to see."""
    c = Call(device, 1, 4, 2, Sq, 400, 64, dtype, INT8, 1)
    power = 110 if dtype == F32 else 8
    c.q = rounded(times_power(c.q, -power), dtype)
    c.k_state[1][:, :, 3:350:7] = times_power(c.k_state[1][:, :, 3:350:7], power)
    c.check(out_dtype=F32)


# ---- weights ------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D, Sq, Skv", [(64, 1, 40), (128, 2, 300), (256, 1, 2000), (64, 40, 65), (128, 130, 300), (256, 40, 200)])
@pytest.mark.parametrize("power", [40, 50, 90, 115])
def test_zero_values_beside_large_ones(device, dtype, D, Sq, Skv, power):
    """Keys whose values are all zero, as a row of zeros is coded, count in the sum of the weights."""
    c = Call(device, 1, 4, 2, Sq, Skv, D, dtype, INT8, 1)
    codes, scales = c.v_state
    codes[:, :, ::2], scales[:, :, ::2] = 0, q8.LEAST_SCALE
    scales[:, :, 1::2] = times_power(scales[:, :, 1::2], power)
    c.check(out_dtype=F32)
    at = Skv - Sq
    c.check(positions_mask(Sq, Skv, [at]), analytic=(True, at, 0), out_dtype=F32)
    codes[:, :, :Skv - 3], scales[:, :, :Skv - 3] = 0, q8.LEAST_SCALE  # all but the last
    c.check(out_dtype=F32)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_many_zero_values(device, dtype):
    """More keys with values of nothing than the largest weight of one fits into f32, in one share, in front of ordinary ones."""
    keys, zeros, D = 300_000, 290_000, 8
    rng = np.random.default_rng(5)
    codes = [rng.integers(-127, 128, (1, 1, keys, D)).astype(np.int8).view(np.uint8) for _ in range(2)]
    scales = [np.full((1, 1, keys), 1 / 127, np.float32) for _ in range(2)]
    codes[1][:, :, :zeros], scales[1][:, :, :zeros] = 0, q8.LEAST_SCALE
    B, Hkv = 16, 32  # units enough that the keys are not shared out
    one = [upload_q8(device, *s, fa.Q8Format.INT8, 1) for s in zip(codes, scales)]
    k, v = (fa.Q8Tensor(t.codes, t.scales, (B, Hkv, keys, D), t.format, 1, (0, 0, t.strides[2]), 0, (0, 0)) for t in one)
    got = upload(device, np.zeros((B, Hkv, 1, D)), dtype).flash_attention(k, v, 1.0, out_dtype=F32).to_numpy().astype(np.float64)
    value = codes[1].view(np.int8).astype(np.float64)[0, 0] * scales[1].astype(np.float64)[0, 0][:, None]
    want, mass = value.sum(0) / keys, np.abs(value).sum(0) / keys
    # weights that are all alike, rounded once (2^-11 at most) times the scale, and sums of so many in f32, a lane's 1 / 16th of them
    assert (np.abs(got - want) <= (2.0 ** -11 + 2.0 ** -24 * keys / 16) * mass).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D, Sq, Skv", [(64, 1, 4000), (64, 40, 3000), (128, 33, 2500), (256, 2, 3000), (64, 40, 60)])
def test_values_near_the_largest(device, dtype, D, Sq, Skv):
    """Values whose sum over a share of the keys is beyond f32, and whose mean is not."""
    c = Call(device, 1, 4, 2, Sq, Skv, D, dtype, INT8, 1)
    c.v_state[0][:] = np.abs(c.v_state[0].view(np.int8)).view(np.uint8)  # (sums do not cancel)
    c.v_state[1][:] = times_power(c.v_state[1], 121)
    c.check(out_dtype=F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D, Sq", [(64, 1), (64, 5), (128, 40), (256, 33)])
@pytest.mark.parametrize("base, step", [(-2.0 ** 24, 2.0 ** 20), (-2.0 ** 30, 2.0 ** 27), (-2.0 ** 100, 2.0 ** 97), (-2.0 ** 127, 2.0 ** 125)])
def test_low_masks_in_their_order(device, dtype, D, Sq, base, step):
    """Rows whose keys a finite mask puts far down weigh those that it puts down the least."""
    Skv = 200
    c = Call(device, 2, 4, 2, Sq, Skv, D, dtype, INT8, 1)
    c.q[:] = 0.0
    m = np.full((Sq, Skv), base, np.float32)
    m[:, 100:] += np.float32(step)
    m[:, 7] = np.finfo(np.float32).min if dtype == F32 else -3.3895314e38
    m[:, 9] = -np.inf
    hidden = np.zeros((1, 1, Sq, Skv), bool)
    hidden[..., :100] = True
    c.check(hidden, mask=(upload(device, m, dtype), fa.MaskKind.QKMask))


# ---- rows that may hold anything ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("anything", [np.inf, -np.inf, np.nan, 3.4e38])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("block", [1, 16])
@pytest.mark.parametrize("Sq", [1, 4, 70])
def test_scales_of_anything_behind_the_last_row(device, anything, dtype, block, Sq):
    lens = [160, 16, 32, 96]
    c = Call(device, len(lens), 4, 2, Sq, 200, 64, dtype, E4M3, block)
    for b, n in enumerate(lens):
        for codes, scales in (c.k_state, c.v_state):
            codes[b, :, n:], scales[b, :, n // block:] = 0x7F, anything
    hidden = np.broadcast_to(np.arange(200) >= np.asarray(lens)[:, None, None, None], (len(lens), 1, Sq, 200))
    got = upload(device, c.q, dtype).flash_attention(*c.tensors(), c.scale, kv_lens=fa.IntTensor(device, lens)).to_numpy()
    for b, n in enumerate(lens):
        for codes, scales in (c.k_state, c.v_state):
            codes[b, :, n:], scales[b, :, n // block:] = 0, 1.0
    c.check(hidden, got=got)


@pytest.mark.parametrize("anything", [np.inf, np.nan])
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("Sq, Skv", [(4, 100), (40, 130)])
def test_scales_of_anything_on_rows_to_come(device, anything, dtype, Sq, Skv):
    """The last key, which only the last query row sees, is nothing to the others."""
    c = Call(device, 1, 4, 2, Sq, Skv, 64, dtype, INT8, 1)
    for state in (c.k_state, c.v_state):
        state[1][:, :, Skv - 1] = anything
    got = upload(device, c.q, dtype).flash_attention(*c.tensors(), c.scale, analytic=(True, Skv - Sq, 0)).to_numpy().astype(np.float64)
    assert not np.isfinite(got[:, :, Sq - 1]).any()
    got[:, :, Sq - 1] = np.nan
    for state in (c.k_state, c.v_state):
        state[1][:, :, Skv - 1] = 1.0
    hidden = positions_mask(Sq, Skv, [Skv - Sq])
    hidden[:, :, Sq - 1] = True
    c.check(hidden, got=got)
