"""A stream that never ends on the framework's sliding cache: KvCache drops its oldest rows, so the text's first tokens are kept beside it, as the prefix, and `sinks`
counts them.  Against the definition over the whole text in 64 bits (context_helpers)."""
import numpy as np
import pytest

import floneum_amd as fa
from context_helpers import definition, rounded, upload, visible

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [fa.F32, fa.F16, fa.BF16])
@pytest.mark.parametrize("B", [1, 3])
@pytest.mark.parametrize("D", [64, 80])
def test_a_stream_that_outlives_its_cache(device, dtype, B, D):
    """A window of 48 keys on a cache of 64: the prompt, single tokens and drafts until the cache has slid several times.  (A batch has to begin alike.)"""
    H, Hkv, sinks, window, room = 4, 2, 4, 48, 64
    rng = np.random.default_rng(D)
    one = lambda *s: rounded(rng.standard_normal(s).astype(np.float32), dtype)  # noqa: E731
    scale = float(np.float32(D ** -0.5))
    cache = fa.KvCache(2, room, dtype, device)
    ks, vs = (np.zeros((B, Hkv, 0, D), np.float32) for _ in range(2))
    prefix = None
    for n in [17] + [1] * 20 + [4] + [1] * 60 + [12] + [1] * 40 + [3, 1, 1]:
        q, k, v = one(B, H, n, D), one(B, Hkv, n, D), one(B, Hkv, n, D)
        new = (k, v)
        if prefix is None:  # the first tokens stay
            k[:, :, :sinks], v[:, :, :sinks] = k[:1, :, :sinks], v[:1, :, :sinks]
            prefix = tuple(upload(device, x[:1, :, :sinks], dtype) for x in (k, v))
            new = (k[:, :, sinks:], v[:, :, sinks:])
        ks, vs = np.concatenate([ks, k], 2), np.concatenate([vs, v], 2)
        own = cache.append(device, *(upload(device, x, dtype) for x in new))
        assert own[0].shape[2] == min(ks.shape[2] - sinks, room) and n + window - 1 <= room
        # the newest row stands behind all keys that are there, whatever was dropped between them and the first tokens
        got = upload(device, q, dtype).flash_attention(*own, scale, analytic=(True, sinks + own[0].shape[2] - n, window), sinks=sinks, prefix=prefix)
        text = ks.shape[2]
        seen = visible(B, n, text - sinks, sinks, offset=text - n, window=window, sinks=sinks)
        want, bound = definition(q, ks[:, :, sinks:], vs[:, :, sinks:], ks[0, :, :sinks], vs[0, :, :sinks], scale, seen, dtype, dtype)
        assert (np.abs(np.asarray(got.to_numpy(), np.float64) - want) <= bound).all(), (n, text)
    assert text > 2 * room
