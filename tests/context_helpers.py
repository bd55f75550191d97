"""Attention over a context in two parts: its definition in 64 bits, and how far a result may be from it."""
import numpy as np

import floneum_amd as fa
from q8_helpers import HALF_STEP, rounded, spread, upload  # noqa: F401

EPS = 2.0 ** -24


def visible(B, Sq, Skv, P, lens=None, positions=None, causal=True, offset=0, window=0, sinks=0):
    """[B, Sq, P + Skv]: which keys a query row sees."""
    key = np.arange(P + Skv)[None, None, :]
    own = np.full(B, Skv) if lens is None else np.clip(np.asarray(lens, np.int64), 0, Skv)
    at = offset + (np.zeros(B, np.int64) if positions is None else np.asarray(positions, np.int64))[:, None, None] + np.arange(Sq)[None, :, None]
    seen = np.broadcast_to(key < P + own[:, None, None], (B, Sq, P + Skv)).copy()
    if causal:
        seen &= key <= at
    if window:
        seen &= (key + window > at) | (key < sinks)
    return seen


def definition(q, k, v, pk, pv, scale, seen, dtype, out_dtype):
    """(result, bound) in 64 bits.  q [B,H,Sq,D], k / v [B,Hkv,Skv,D], pk / pv [Hkv,P,D] (hidden rows may hold anything).

    The bound counts, per output element with mass = sum of p |v| over the row:
      output           half a step of the output's type
      scores           a sum of D products in f32 (D roundings at most, of at most the sum of the products' magnitudes), the scale, its product
                       with log2 e and the subtraction of the reference: 8 roundings of the largest score or reference; f32 tensors go
                       through bf16 terms whose dropped products are below 4 steps of a product; both numerator and denominator have them
      weights          half a step of the tensors' type for the second product (f32: 4 steps, three terms), 2^-22 for exp2
      small weights    f16 weights below 2^-14 of the reference have a fixed step: 2^-25 of the largest weight each
      sums             n / 16 additions one after the other (a matrix instruction adds 16 keys or more), 64 where shares are joined"""
    B, H, Sq, D = q.shape
    P = pk.shape[1]
    group = H // k.shape[1] if k.shape[1] else 1
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b in range(B):
        used = seen[b].any(0)
        for h in range(H):
            g = h // group
            kk = np.where(used[:, None], np.concatenate([pk[g], k[b, g]]).astype(np.float64), 0.0)
            vv = np.where(used[:, None], np.concatenate([pv[g], v[b, g]]).astype(np.float64), 0.0)
            x = q[b, h].astype(np.float64)
            s = np.where(seen[b], x @ kk.T * scale, -np.inf)
            top = s.max(-1, keepdims=True, initial=-np.inf)
            with np.errstate(invalid="ignore", divide="ignore"):
                w = np.exp(s - top)
                p = w / w.sum(-1, keepdims=True)
            out[b, h] = p @ vv
            n = max(int(seen[b].sum(-1).max(initial=0)), 1)
            # a row's largest sum of products; its largest score bounds the reference
            reach = (np.where(seen[b], np.abs(x) @ np.abs(kk).T, 0.0).max(-1, keepdims=True, initial=0.0)) * abs(scale)
            score = EPS * (D + 4 * (dtype == fa.F32)) * reach + EPS * 8 * np.log2(np.e) * np.abs(np.where(np.isfinite(top), top, 0.0)) + EPS * 8
            score = score + EPS * 8 * np.where(seen[b] & (p > 0), np.abs(np.where(seen[b], s, 0.0)), 0.0).max(-1, keepdims=True, initial=0.0)
            weight = (HALF_STEP[dtype] if dtype != fa.F32 else 8 * EPS) + 2.0 ** -22
            sums = EPS * (n / 16 + 64)
            mass = np.nan_to_num(p) @ np.abs(vv)
            small = 2.0 ** -25 * np.nan_to_num(p).max(-1, keepdims=True, initial=0.0) * (seen[b].astype(np.float64) @ np.abs(vv)) * (dtype == fa.F16)
            bound[b, h] = HALF_STEP[out_dtype] * np.abs(out[b, h]) + (2 * score + weight + 2 * sums) * mass + small + 1e-30
    return out, bound


class Call:
    """A call on the device and its definition, from one seed."""

    def __init__(self, device, dtype, B, H, Hkv, Sq, Skv, P, D, seed=0, scale=None, std=1.0, lean=0.7):
        rng = np.random.default_rng(seed)
        self.device, self.dtype, self.shape, self.P = device, dtype, (B, H, Sq, D), P
        self.scale = float(np.float32(D ** -0.5 if scale is None else scale))
        one = lambda *s: rounded(rng.standard_normal(s).astype(np.float32) * np.float32(std), dtype)  # noqa: E731
        self.q, self.k, self.v, self.pk, self.pv = one(B, H, Sq, D), one(B, Hkv, Skv, D), one(B, Hkv, Skv, D), one(Hkv, P, D), one(Hkv, P, D)
        # the first keys draw weight, as first tokens do
        first = self.pk if P else self.k
        first[..., :3, :] = rounded(first[..., :3, :] + np.float32(lean) * self.q[:1, :1, :1].mean((0, 1, 2)), dtype)
        self.Skv = Skv

    def mask(self, **how):
        return visible(self.shape[0], self.shape[2], self.Skv, self.P, **how)

    def run(self, lens=None, positions=None, causal=True, offset=0, window=0, sinks=0, out_dtype=None, out=None, tensors=None, poison=False):
        """The device's result (f32); `poison`: rows that no query row sees hold NaN."""
        d = self.device
        q, k, v, pk, pv = self.q, self.k, self.v, self.pk[None], self.pv[None]
        if poison:
            seen = self.mask(lens=lens, positions=positions, causal=causal, offset=offset, window=window, sinks=sinks)
            k, v, pk, pv = k.copy(), v.copy(), pk.copy(), pv.copy()
            for b in range(self.shape[0]):
                k[b][:, ~seen[b].any(0)[self.P:]] = np.nan
                v[b][:, ~seen[b].any(0)[self.P:]] = np.nan
            pk[0][:, ~seen.any((0, 1))[:self.P]] = np.nan
            pv[0][:, ~seen.any((0, 1))[:self.P]] = np.nan
        if tensors is None:
            tensors = [upload(d, x, self.dtype) for x in (q, k, v, pk, pv)]
        tq, tk, tv, tpk, tpv = tensors
        got = tq.flash_attention(tk, tv, self.scale, analytic=(causal, offset, window) if causal or window else None, sinks=sinks,
                                 prefix=(tpk, tpv) if self.P else None, kv_lens=None if lens is None else fa.IntTensor(d, np.asarray(lens, np.int32)),
                                 q_positions=None if positions is None else fa.IntTensor(d, np.asarray(positions, np.int32)),
                                 out_dtype=out_dtype, out=out)
        return np.asarray(got.to_numpy(), np.float32)

    def check(self, got, out_dtype=None, **how):
        seen = self.mask(**how)
        want, bound = definition(self.q, self.k, self.v, self.pk, self.pv, self.scale, seen, self.dtype, self.dtype if out_dtype is None else out_dtype)
        none = ~seen.any(-1)[:, None, :, None] & np.ones(want.shape, bool)
        assert np.isnan(got[none]).all(), "rows without a key are NaN"
        off = np.abs(got.astype(np.float64) - want)
        assert not np.isnan(got[~none]).any(), "NaN in a row that sees keys"
        worst = np.unravel_index(np.argmax(np.where(none, 0, off / bound)), off.shape) if off.size else None
        assert off.size == 0 or (off[~none] <= bound[~none]).all(), (worst, got[worst], want[worst], bound[worst])

    def both(self, out_dtype=None, poison=True, **how):
        self.check(self.run(out_dtype=out_dtype, poison=poison, **how), out_dtype, **how)
