"""Attention over a context in two parts on the tiled kernels: calls of more than 256 rows times heads of a group, which no other kernel takes unless
the tiled ones refuse.  Against the definition in 64 bits (context_helpers)."""
import ctypes

import numpy as np
import pytest

import floneum_amd as fa
from context_helpers import Call, definition, rounded, spread, upload

pytestmark = pytest.mark.gpu
TYPES = [fa.F32, fa.F16, fa.BF16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 40, 64, 72, 80, 96, 104, 128, 136, 160, 200, 256])
@pytest.mark.parametrize("B, H, Hkv, Sq, Skv, window, sinks", [(2, 4, 2, 140, 517, 129, 5), (1, 3, 1, 100, 333, 64, 70), (1, 2, 2, 300, 301, 1, 1)])
def test_sinks(device, dtype, D, B, H, Hkv, Sq, Skv, window, sinks):
    Call(device, dtype, B, H, Hkv, Sq, Skv, 0, D, seed=D).both(offset=Skv - Sq, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("B, H, Hkv, Sq, Skv, P", [(2, 2, 1, 133, 150, 200), (3, 6, 1, 50, 70, 129), (2, 3, 1, 90, 90, 513)])
def test_prefix(device, dtype, D, B, H, Hkv, Sq, Skv, P):
    lens = np.random.default_rng(P).integers(Sq, Skv + 1, B)
    Call(device, dtype, B, H, Hkv, Sq, Skv, P, D, seed=D).both(lens=lens, positions=lens - Sq, offset=P)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window, sinks", [(100, 4), (300, 260), (20, 1), (1, 0), (5, 5), (450, 300)])
def test_prefix_window_sinks(device, dtype, D, window, sinks):
    lens = np.asarray([160, 200, 150])
    Call(device, dtype, 3, 4, 2, 150, 200, 250, D, seed=1).both(lens=lens, positions=lens - 150, offset=250, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 160])
def test_rows_without_a_key(device, dtype, D):
    c = Call(device, dtype, 5, 4, 2, 140, 90, 0, D, seed=3)
    c.both(lens=[0, -5, 90, 1000, 1], positions=[0, 0, -200, 5, 0], offset=50, window=30, sinks=2)
    c.both(lens=[0, -5, 90, 1000, 1], positions=[0, 0, -200, 5, 0], offset=50)
    c = Call(device, dtype, 3, 4, 2, 140, 90, 33, D, seed=3)
    c.both(lens=[0, -5, 90], positions=[-1000, 0, 30], offset=20, window=7, sinks=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [128, 256])
def test_without_a_causal_mask(device, dtype, D):
    Call(device, dtype, 2, 4, 2, 140, 90, 130, D).both(causal=False)
    Call(device, dtype, 2, 4, 2, 140, 90, 130, D).both(causal=False, offset=150, window=20, sinks=9)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window, sinks", [(0, 0), (200, 3), (1000, 40), (64, 128), (31, 33)])
@pytest.mark.parametrize("D", [64, 256])
def test_positions_over_the_prefix(device, dtype, window, sinks, D):
    c = Call(device, dtype, 6, 4, 2, 140, 220, 700, D, seed=2)
    c.both(lens=[220, 150, 0, 177, 220, 1], positions=[0, 40, 300, 650, 735, 690], offset=5, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 192])
def test_layouts(device, dtype, D):
    c = Call(device, dtype, 2, 4, 2, 140, 250, 70, D, seed=1)
    how = dict(offset=70 + 250 - 140, window=90, sinks=3)
    values = [c.q, c.k, c.v, c.pk[None], c.pv[None]]
    for order in ([0, 2, 1, 3], [1, 2, 0, 3], [3, 0, 1, 2]):
        c.check(c.run(tensors=[upload(device, x, dtype, order) for x in values], **how), **how)
    for steps in ([1, 1, 2, 1], [1, 2, 1, 1], [1, 1, 1, 2]):
        whole, out = spread(device, c.shape, dtype, steps, 7.0)
        c.check(c.run(out=out, **how), **how)
        left = np.ones(whole.shape, bool)
        left[tuple(slice(None, None, s) for s in steps)] = False
        assert np.unique(whole.to_numpy()[left]).size <= 1  # nothing is written beside the result
    tensors = []
    for x, steps in zip(values, ((2, 1, 3, 1), (1, 2, 2, 1), (1, 1, 3, 1), (1, 1, 4, 1), (1, 3, 1, 1))):
        host = np.full([n * s for n, s in zip(x.shape, steps)], 5.0, np.float32)
        host[tuple(slice(None, None, s) for s in steps)] = x
        strides = [st * s for st, s in zip(spread(device, x.shape, dtype, steps, 0.0)[0].strides, steps)]
        tensors.append(fa.Tensor(upload(device, host, dtype).buffer, dtype, x.shape, strides))
    c.check(c.run(tensors=tensors, **how), **how)


@pytest.mark.parametrize("dtype", [fa.F16, fa.BF16])
@pytest.mark.parametrize("D", [128, 256])
def test_f32_results(device, dtype, D):
    Call(device, dtype, 2, 4, 2, 140, 150, 70, D).both(out_dtype=fa.F32, offset=80, window=90, sinks=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 3.0])
@pytest.mark.parametrize("D", [64, 192])
def test_scales(device, dtype, scale, D):
    Call(device, dtype, 2, 4, 2, 140, 150, 70, D, scale=scale).both(offset=80, window=90, sinks=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Skv, P", [(200, 0), (200, 130)])
@pytest.mark.parametrize("D", [64, 128, 192])
def test_infinite_elements(device, dtype, Skv, P, D):
    """A key whose score is -inf has no weight; an infinite value of a key that every row sees makes its dim infinite, and no other."""
    Sq = 140
    c = Call(device, dtype, 2, 4, 2, Sq, Skv, P, D, seed=8)
    c.q[..., 0] = np.abs(c.q[..., 0]) + rounded(np.float32(0.25), dtype)
    first = (c.pk[None], c.pv[None]) if P else (c.k, c.v)
    first[0][:, :, 7, 0] = -np.inf
    first[1][:, 0, 5, 3], first[1][:, 1, 2, D - 1] = np.inf, -np.inf
    got = c.run(offset=P + Skv - Sq)
    dims = [np.arange(D) != d for d in (3, D - 1)]
    for h in range(4):
        assert (got[:, h, :, ~dims[h // 2]] == (np.inf, -np.inf)[h // 2]).all()
    first[0][:, :, 7, 0] = 0.0
    first[1][:, 0, 5, 3] = first[1][:, 1, 2, D - 1] = 0.0
    seen = c.mask(offset=P + Skv - Sq)
    seen[:, :, 7] = False
    want, bound = definition(c.q, c.k, c.v, c.pk, c.pv, c.scale, seen, dtype, dtype)
    for h in range(4):
        off = np.abs(got[:, h][..., dims[h // 2]] - want[:, h][..., dims[h // 2]])
        assert (off <= bound[:, h][..., dims[h // 2]]).all()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window, sinks", [(0, 0), (100, 20)])
def test_f32_beyond_bf16(device, D, window, sinks):
    """Finite f32 elements that no sum of finite bf16 terms makes, where a row meets them times zero, beside values of 3.4e38 that few rows see."""
    c = Call(device, fa.F32, 2, 4, 2, 140, 200, 130, D, seed=8)
    c.q[..., 1] = 0.0
    c.pk[:, 11, 1] = c.k[:, :, 3, 1] = 3.4e38
    c.k[:, :, 190, 1] = -3.4e38  # of the last rows alone
    how = dict(offset=190, window=window, sinks=sinks)
    got = c.run(**how)
    c.pk[:, 11, 1] = c.k[:, :, 3, 1] = c.k[:, :, 190, 1] = 0.0
    c.check(got, **how)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 256])
def test_large_scores(device, dtype, D):
    for window, sinks in ((0, 0), (60, 2)):
        Call(device, dtype, 2, 4, 2, 140, 190, 130, D, seed=9, scale=1.0, std=8.0).both(offset=180, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_a_captured_prompt(device, dtype, D):
    """Recorded once, replayed with other queries, lengths and positions; eager calls on the same workspace between the replays."""
    B, H, Hkv, Sq, Skv, P = 3, 4, 1, 70, 300, 500
    c = Call(device, dtype, B, H, Hkv, Sq, Skv, P, D, seed=11)
    tensors = [upload(device, x, dtype) for x in (c.q, c.k, c.v, c.pk[None], c.pv[None])]
    lens, at = fa.IntTensor(device, [Sq] * B), fa.IntTensor(device, [0] * B)
    outs = [upload(device, np.zeros(c.shape), dtype) for _ in range(2)]

    def write(t, host):
        host = np.ascontiguousarray(host)
        fa.check(fa.lib().fhip_memcpy_h2d(device.stream, ctypes.c_void_p(t.buffer.ptr), host.ctypes.data_as(ctypes.c_void_p), host.nbytes))

    def step():
        for o, (window, sinks) in zip(outs, ((0, 0), (400, 5))):
            tensors[0].flash_attention(*tensors[1:3], c.scale, analytic=(True, P, window), sinks=sinks, prefix=tuple(tensors[3:]), kv_lens=lens,
                                       q_positions=at, out=o)

    step()
    device.synchronize()
    with device.capture() as cap:
        step()
    rng = np.random.default_rng(13)
    for turn in range(4):
        n = np.asarray([Skv, int(rng.integers(Sq, Skv)), Sq], np.int32)
        write(lens, n)
        write(at, n - Sq)
        for o in outs:
            fa.check(fa.lib().fhip_memset(device.stream, ctypes.c_void_p(o.buffer.ptr), 0x7F, o.buffer.nbytes))
        device.synchronize()
        cap.graph.launch()
        replayed = [np.asarray(o.to_numpy(), np.float32) for o in outs]
        c.check(replayed[0], lens=n, positions=n - Sq, offset=P)
        c.check(replayed[1], lens=n, positions=n - Sq, offset=P, window=400, sinks=5)
        step()
        for x, o in zip(replayed, outs):
            assert np.array_equal(x, np.asarray(o.to_numpy(), np.float32))
