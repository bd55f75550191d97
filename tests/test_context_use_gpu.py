"""Attention over a context in two parts as a program uses it: every kernel that a call can reach, recorded steps, streams, workspaces, long
caches, elements that are not finite, a conversation from its prompt on.  Against the definition in 64 bits (context_helpers)."""
import ctypes

import numpy as np
import pytest

import floneum_amd as fa
from context_helpers import Call, definition, rounded, spread, upload, visible

pytestmark = pytest.mark.gpu
TYPES = [fa.F32, fa.F16, fa.BF16]


def write(device, t, host):
    """host's bytes into the tensor or buffer t, on the device's stream."""
    host = np.ascontiguousarray(host)
    fa.check(fa.lib().fhip_memcpy_h2d(device.stream, ctypes.c_void_p(t.buffer.ptr), host.ctypes.data_as(ctypes.c_void_p), host.nbytes))


# ---- kernels -----------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, H, Hkv, Sq, Skv, P, D", [
    (128, 8, 1, 1, 20, 4100, 64),    # 1024 rows on the prefix, in shares of its keys; own keys in the kernel for few rows
    (40, 16, 1, 1, 0, 4100, 128),    # the same without own keys
    (2, 16, 1, 3, 20, 4100, 128),    # 96 rows
    (3, 3, 1, 43, 60, 1000, 72),     # 129 rows of a unit, three heads of a group: head_dim below the kernel's
    (6, 16, 1, 4, 33, 2100, 256),    # 384 rows
    (3, 8, 1, 7, 33, 2100, 192),
    (3, 4, 1, 20, 0, 300, 64), (3, 4, 1, 20, 0, 300, 192), (3, 4, 1, 70, 0, 300, 64),  # no own keys, in the tiled kernels
    (2, 5, 1, 60, 60, 300, 160),     # 300 rows of a unit: both parts in launches of their own above head_dim 128
])
def test_rows_of_all_sequences_on_the_prefix(device, dtype, B, H, Hkv, Sq, Skv, P, D):
    rng = np.random.default_rng(P + B)
    lens = rng.integers(Sq, Skv + 1, B) if Skv else None
    Call(device, dtype, B, H, Hkv, Sq, Skv, P, D, seed=D).both(lens=lens, positions=None if lens is None else lens - Sq, offset=P, causal=Skv > 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H, Hkv, Sq, D", [(4, 1, 65, 128), (4, 1, 257, 64), (2, 1, 130, 256), (1, 1, 129, 80), (3, 1, 87, 96), (4, 2, 321, 128), (8, 1, 40, 128)])
def test_last_rows_apart(device, dtype, H, Hkv, Sq, D):
    """Rows that fill workgroups but for a few, in batches that fill the device: the few run on their own."""
    B = 40
    c = Call(device, dtype, B, H, Hkv, Sq, Sq + 9, 130, D, seed=Sq)
    lens = np.random.default_rng(Sq).integers(Sq, Sq + 10, B)
    c.both(lens=lens, positions=lens - Sq, offset=130)
    c.both(offset=139, window=100, sinks=7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Sq, Skv, P, window, sinks", [
    (300, 3000, 0, 700, 70),   # first tokens of more than a tile, keys in shares
    (70, 900, 900, 1200, 3),   # the window lies over both parts
    (70, 200, 2000, 150, 2100),  # first tokens reach into the sequences' own keys
    (64, 64, 640, 64, 64), (65, 65, 63, 1, 1), (200, 200, 1, 5, 1),
])
def test_prompts_under_a_window(device, dtype, D, Sq, Skv, P, window, sinks):
    Call(device, dtype, 2, 6, 2, Sq, Skv, P, D, seed=Sq).both(offset=P + Skv - Sq, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 40])
@pytest.mark.parametrize("window, sinks", [(0, 0), (200, 3), (1000, 40), (64, 128), (31, 33)])
def test_positions_over_the_prefix(device, dtype, Sq, window, sinks):
    """Sequences whose rows stand anywhere, in the prefix too: each sees its own run of it."""
    c = Call(device, dtype, 6, 4, 2, Sq, 120, 700, 64, seed=2)
    c.both(lens=[120, 50, 0, 77, 120, 1], positions=[0, 40, 300, 650, 735, 690], offset=5, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [16, 40, 104, 136, 200, 248])
def test_other_head_dims(device, dtype, D):
    for Sq in (1, 50):
        Call(device, dtype, 3, 4, 2, Sq, 80, 150, D, seed=D).both(offset=230 - Sq, window=140, sinks=5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H, Hkv", [(5, 1), (7, 7), (12, 4), (33, 1), (40, 2)])
def test_groups(device, dtype, H, Hkv):
    """Groups that divide no tile, and such as fill more than one block of columns by themselves."""
    for Sq in (1, 2, 37):
        lens = np.asarray([90, Sq])
        Call(device, dtype, 2, H, Hkv, Sq, 90, 60, 64, seed=H).both(lens=lens, positions=lens - Sq, offset=60, window=70, sinks=2)


# ---- memory ------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [fa.F16, fa.F32])
@pytest.mark.parametrize("Sq", [1, 40])
def test_rows_behind_32_bits(device, dtype, Sq):
    """A cache of 2^32 elements and more, as the sequence's own and as the prefix: first tokens at its start, the window at its end."""
    D, rows, window, sinks = 64, (1 << 26) + 5000, 300, 4
    n = window + Sq
    c = Call(device, dtype, 1, 4, 1, Sq, n + sinks, 0, D, seed=4)
    big = [fa.Tensor.empty(device, (1, 1, rows, D), dtype) for _ in range(2)]
    size = 4 if dtype == fa.F32 else 2
    for t, x in zip(big, (c.k, c.v)):
        for first, part in ((0, x[:, :, :sinks]), (rows - n, x[:, :, sinks:])):
            part = np.ascontiguousarray(part, np.float32 if dtype == fa.F32 else np.float16)
            at = ctypes.c_void_p(t.buffer.ptr + first * D * size)
            fa.check(fa.lib().fhip_memcpy_h2d(device.stream, at, part.ctypes.data_as(ctypes.c_void_p), part.nbytes))
    q = upload(device, c.q, dtype)
    how = dict(offset=sinks + n - Sq, window=window, sinks=sinks)  # of the definition, on the rows that are visible alone
    got = q.flash_attention(*big, c.scale, analytic=(True, rows - Sq, window), sinks=sinks).to_numpy()
    c.check(np.asarray(got, np.float32), **how)
    none = fa.Tensor.empty(device, (1, 1, 0, D), dtype)
    got = q.flash_attention(none, none, c.scale, analytic=(True, rows - Sq, window), sinks=sinks, prefix=big).to_numpy()
    c.check(np.asarray(got, np.float32), **how)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 9])
def test_rows_far_apart(device, dtype, Sq):
    """Rows 2^25 bytes apart and more."""
    D, rows, size = 64, 37, 4 if dtype == fa.F32 else 2
    step = ((1 << 25) + 4096) // size
    c = Call(device, dtype, 1, 4, 1, Sq, rows, 0, D, seed=5)
    tensors = []
    for x in (c.k, c.v):
        b = fa.Buffer(device, rows * step * size)
        for r in range(rows):
            part = fa.Tensor.from_numpy(device, np.ascontiguousarray(x[0, 0, r], np.float32), dtype)
            fa.check(fa.lib().fhip_memcpy_d2d(device.stream, ctypes.c_void_p(b.ptr + r * step * size), ctypes.c_void_p(part.buffer.ptr), D * size))
        tensors.append(fa.Tensor(b, dtype, (1, 1, rows, D), (rows * step, rows * step, step, 1)))
    how = dict(offset=rows - Sq, window=20, sinks=2)
    q = upload(device, c.q, dtype)
    c.check(np.asarray(q.flash_attention(*tensors, c.scale, analytic=(True, rows - Sq, 20), sinks=2).to_numpy(), np.float32), **how)
    none = fa.Tensor.empty(device, (1, 1, 0, D), dtype)
    c.check(np.asarray(q.flash_attention(none, none, c.scale, analytic=(True, rows - Sq, 20), sinks=2, prefix=tensors).to_numpy(), np.float32), **how)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 40])
def test_strided_parts(device, dtype, Sq):
    """Own keys, values and both halves of the prefix at rows of different lengths, a result whose heads lie behind its rows, a padded batch whose last
    sequences are left out."""
    B, H, Hkv, Skv, P, D = 3, 4, 2, 90, 70, 64
    c = Call(device, dtype, B, H, Hkv, Sq, Skv, P, D, seed=6)
    tensors = []
    for x, steps in ((c.q, (2, 1, 3, 1)), (c.k, (1, 2, 2, 1)), (c.v, (1, 1, 3, 1)), (c.pk[None], (1, 1, 4, 1)), (c.pv[None], (1, 3, 1, 1))):
        whole, t = spread(device, x.shape, dtype, steps, 5.0)
        host = np.full(whole.shape, 5.0, np.float32)
        host[tuple(slice(None, None, s) for s in steps)] = x
        tensors.append(fa.Tensor(upload(device, host, dtype).buffer, dtype, t.shape, t.strides))
    whole = upload(device, np.full((B + 2, Sq, H, D), 7.0), dtype)
    out = fa.Tensor(whole.buffer, dtype, (B, Sq, H, D), whole.strides).transpose(1, 2)
    lens = [90, 41, Sq]
    c.check(c.run(tensors=tensors, out=out, lens=lens, positions=np.subtract(lens, Sq), offset=P), lens=lens, positions=np.subtract(lens, Sq), offset=P)
    assert (np.asarray(whole.to_numpy(), np.float32)[B:] == 7.0).all()


def args_of(device, c, q, k, v, pk, pv, out, offset):
    a = fa.CContextAttnArgs()
    a.q, a.out, a.k, a.v, a.prefix_k, a.prefix_v = (t._c4() for t in (q, out, k, v, pk, pv))
    a.dtype = a.out_dtype = c.dtype
    a.scale, a.causal, a.q_pos_offset = c.scale, 1, offset
    return a


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, H, Sq, Skv, P", [(2, 8, 1, 2000, 500), (30, 8, 1, 20, 2000), (3, 4, 100, 300, 700), (40, 4, 65, 65, 300)])
def test_workspaces(device, dtype, B, H, Sq, Skv, P):
    """Too small, absent or unaligned ones are refused; one that starts with anything serves, and nothing behind it is written."""
    c = Call(device, dtype, B, H, 2, Sq, Skv, P, 64, seed=7)
    t = [upload(device, x, dtype) for x in (c.q, c.k, c.v, c.pk[None], c.pv[None])]
    out = fa.Tensor.empty(device, c.shape, dtype)
    a = args_of(device, c, *t, out, P + Skv - Sq)
    need = ctypes.c_size_t()
    L = fa.lib()
    fa.check(L.fhip_context_attention_workspace_bytes(ctypes.byref(a), device.compute_units, ctypes.byref(need)))
    memory = fa.Buffer(device, need.value + 4096)
    if need.value:
        for ptr, size in ((None, 0), (memory.ptr, need.value - 1), (memory.ptr + 4, need.value)):
            a.workspace, a.workspace_bytes = ptr, size
            assert L.fhip_context_attention(device.stream, ctypes.byref(a)) == fa.ERR_WORKSPACE
    a.workspace, a.workspace_bytes = memory.ptr, need.value
    for fill in (0, 0xFF, 0x55):
        fa.check(L.fhip_memset(device.stream, ctypes.c_void_p(memory.ptr), fill, need.value + 4096))
        assert L.fhip_context_attention(device.stream, ctypes.byref(a)) == fa.OK
        c.check(np.asarray(out.to_numpy(), np.float32), offset=P + Skv - Sq)
        behind = np.empty(4096, np.uint8)
        fa.check(L.fhip_memcpy_d2h(device.stream, behind.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(memory.ptr + need.value), 4096))
        assert (behind == fill).all()


# ---- elements that are not finite --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq, Skv, P", [(1, 300, 0), (1, 40, 200), (40, 90, 0), (40, 90, 130)])
@pytest.mark.parametrize("D", [64, 128, 192])
def test_infinite_elements(device, dtype, Sq, Skv, P, D):
    """A key whose score is -inf has no weight; an infinite value of a key that every row sees makes its dim infinite, and no other."""
    c = Call(device, dtype, 2, 4, 2, Sq, Skv, P, D, seed=8)
    c.q[..., 0] = np.abs(c.q[..., 0]) + rounded(np.float32(0.25), dtype)
    first = (c.pk[None], c.pv[None]) if P else (c.k, c.v)
    first[0][:, :, 7, 0] = -np.inf
    first[1][:, 0, 5, 3], first[1][:, 1, 2, D - 1] = np.inf, -np.inf
    how = dict(offset=P + Skv - Sq)
    got = c.run(**how)
    dims = [np.arange(D) != d for d in (3, D - 1)]
    for h in range(4):
        assert (got[:, h, :, ~dims[h // 2]] == (np.inf, -np.inf)[h // 2]).all()
    # the other dims: the key at -inf hidden, the infinite values zero
    first[0][:, :, 7, 0] = 0.0
    first[1][:, 0, 5, 3] = first[1][:, 1, 2, D - 1] = 0.0
    seen = c.mask(**how)
    seen[:, :, 7] = False
    want, bound = definition(c.q, c.k, c.v, c.pk, c.pv, c.scale, seen, dtype, dtype)
    for h in range(4):
        off = np.abs(got[:, h][..., dims[h // 2]] - want[:, h][..., dims[h // 2]])
        assert (off <= bound[:, h][..., dims[h // 2]]).all()


@pytest.mark.parametrize("Sq", [1, 40])
def test_f32_beyond_bf16(device, Sq):
    """Finite f32 elements that no sum of finite bf16 terms makes, where a row meets them times zero."""
    c = Call(device, fa.F32, 2, 4, 2, Sq, 90, 130, 64, seed=8)
    c.q[..., 1] = 0.0
    c.pk[:, 11, 1] = c.k[:, :, 3, 1] = 3.4e38
    seen = c.mask(offset=220 - Sq)
    got = c.run(offset=220 - Sq)
    c.pk[:, 11, 1] = c.k[:, :, 3, 1] = 0.0
    want, bound = definition(c.q, c.k, c.v, c.pk, c.pv, c.scale, seen, fa.F32, fa.F32)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 40])
def test_large_scores(device, dtype, Sq):
    """Scores of some thousands: one key takes all the weight, and no exponential overflows."""
    Call(device, dtype, 2, 4, 2, Sq, 90, 130, 64, seed=9, scale=1.0, std=12.0).both(offset=220 - Sq)
    Call(device, dtype, 2, 4, 2, Sq, 90, 130, 64, seed=9, scale=1.0, std=12.0).both(offset=220 - Sq, window=60, sinks=2)


# ---- calls beside and after each other -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("with_native", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_both_ways_to_the_library(device, monkeypatch, dtype, with_native):
    """The mirror's calls through its native half and through ctypes."""
    assert fa._native is not None
    if not with_native:
        monkeypatch.setattr(fa, "_native", None)
    lens = np.asarray([60, 200])
    for Sq in (1, 40):
        c = Call(device, dtype, 2, 4, 2, Sq, 200, 250, 64, seed=Sq)
        c.both(lens=lens, positions=lens - Sq, offset=250, window=100, sinks=4)
        c.both(lens=lens, positions=lens - Sq, offset=250)
        c.both(out_dtype=fa.F32, causal=False)
        got = upload(device, c.q, dtype).flash_attention(*(upload(device, x, dtype) for x in (c.k, c.v)), c.scale, sinks=np.int64(3),
                                                         analytic=fa.CAnalyticMask(1, 1, 200 - Sq, 50))
        c.pk, c.pv, c.P = c.pk[:, :0], c.pv[:, :0], 0
        c.check(np.asarray(got.to_numpy(), np.float32), offset=200 - Sq, window=50, sinks=3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 4, 70])
def test_a_captured_step(device, dtype, Sq):
    """Recorded once, replayed with other queries, lengths and positions in device memory; eager calls on the same workspace between the replays."""
    B, H, Hkv, Skv, P, D = 3, 8, 2, 300, 500, 64
    c = Call(device, dtype, B, H, Hkv, Sq, Skv, P, D, seed=11)
    tensors = [upload(device, x, dtype) for x in (c.q, c.k, c.v, c.pk[None], c.pv[None])]
    lens, at, out = fa.IntTensor(device, [Sq] * B), fa.IntTensor(device, [0] * B), upload(device, np.zeros(c.shape), dtype)
    outs = [out, upload(device, np.zeros(c.shape), dtype)]

    def step():
        for o, (window, sinks) in zip(outs, ((0, 0), (400, 5))):
            tensors[0].flash_attention(*tensors[1:3], c.scale, analytic=(True, P, window), sinks=sinks, prefix=tensors[3:], kv_lens=lens, q_positions=at, out=o)

    step()
    device.synchronize()
    with device.capture() as cap:
        step()
    other = Call(device, dtype, 2, 8, 2, 1, 4000, 0, 128, seed=12)
    rng = np.random.default_rng(13)
    for turn in range(4):
        c.q = rounded(rng.standard_normal(c.shape).astype(np.float32), dtype)
        write(device, tensors[0], upload(device, c.q, dtype).to_numpy() if dtype != fa.BF16 else (c.q.view(np.uint32) >> 16).astype(np.uint16))
        n = [Skv, int(rng.integers(Sq, Skv)), Sq]
        write(device, lens, np.asarray(n, np.int32))
        write(device, at, np.asarray(n, np.int32) - Sq)
        for o in outs:
            fa.check(fa.lib().fhip_memset(device.stream, ctypes.c_void_p(o.buffer.ptr), 0x7F, o.buffer.nbytes))
        device.synchronize()
        cap.graph.launch()
        replayed = [np.asarray(o.to_numpy(), np.float32) for o in outs]
        how = dict(lens=n, positions=np.subtract(n, Sq), offset=P)
        c.check(replayed[0], **how)
        c.check(replayed[1], window=400, sinks=5, **how)
        other.both(offset=3999, window=1000, sinks=4)
        step()
        for x, o in zip(replayed, outs):
            assert np.array_equal(x, np.asarray(o.to_numpy(), np.float32))


@pytest.mark.parametrize("dtype", TYPES)
def test_two_streams(device, dtype):
    """The same calls on two streams of one device at once, each with its own workspace."""
    other = device.with_new_stream()
    for Sq, B in ((1, 4), (1, 70), (70, 2)):
        calls = [Call(dev, dtype, B, 8, 2, Sq, 600, 900, 64, seed=s) for s, dev in enumerate((device, other))]
        inputs = [[upload(c.device, x, dtype) for x in (c.q, c.k, c.v, c.pk[None], c.pv[None])] for c in calls]
        outs = [[], []]
        for _ in range(5):
            for i, t in enumerate(inputs):
                outs[i].append(t[0].flash_attention(*t[1:3], calls[i].scale, analytic=(True, 1500 - Sq, 700), sinks=3, prefix=t[3:]))
        for c, got in zip(calls, outs):
            first = np.asarray(got[0].to_numpy(), np.float32)
            assert all(np.array_equal(first, np.asarray(x.to_numpy(), np.float32)) for x in got)  # (and every call gives the same bits)
            c.check(first, offset=1500 - Sq, window=700, sinks=3)


# ---- a conversation ------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
def test_conversations_behind_one_instruction(device, dtype):
    """A shared instruction goes through one cache as a prompt of its own; then a batch of answers grows behind it, row by row and in a draft, each step's
    keys appended to the sequences' cache: over the whole context, and under a window whose first tokens stay visible."""
    B, H, Hkv, D, P, window, sinks = 3, 4, 2, 64, 150, 60, 4
    rng = np.random.default_rng(14)
    one = lambda *s: rounded(rng.standard_normal(s).astype(np.float32), dtype)  # noqa: E731
    scale = float(np.float32(D ** -0.5))
    shared, own = fa.KvCache(2, 4096, dtype, device), fa.KvCache(2, 4096, dtype, device)
    q, k, v = one(1, H, P, D), one(1, Hkv, P, D), one(1, Hkv, P, D)
    prefix = shared.append(device, *(upload(device, x, dtype) for x in (k, v)))
    got = upload(device, q, dtype).flash_attention(*prefix, scale, analytic=(True, 0, window), sinks=sinks).to_numpy()
    none = np.zeros((Hkv, 0, D), np.float32)
    want, bound = definition(q, k, v, none, none, scale, visible(1, P, P, 0, window=window, sinks=sinks), dtype, dtype)
    assert (np.abs(np.asarray(got, np.float64) - want) <= bound).all()
    pk, pv = k[0], v[0]
    ks, vs = (np.zeros((B, Hkv, 0, D), np.float32) for _ in range(2))
    for n in [9] + [1] * 6 + [4] + [1] * 3 + [45]:
        q, k, v = one(B, H, n, D), one(B, Hkv, n, D), one(B, Hkv, n, D)
        keys = own.append(device, *(upload(device, x, dtype) for x in (k, v)))
        at = ks.shape[2]
        ks, vs = np.concatenate([ks, k], 2), np.concatenate([vs, v], 2)
        for w, s in ((0, 0), (window, sinks)):
            got = upload(device, q, dtype).flash_attention(*keys, scale, analytic=(True, P + at, w), sinks=s, prefix=prefix).to_numpy()
            want, bound = definition(q, ks, vs, pk, pv, scale, visible(B, n, at + n, P, offset=P + at, window=w, sinks=s), dtype, dtype)
            assert (np.abs(np.asarray(got, np.float64) - want) <= bound).all(), (n, at, w)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 40, 300])
def test_a_prefix_of_no_rows(device, dtype, Sq):
    c = Call(device, dtype, 2, 4, 2, Sq, 350, 0, 64, seed=15)
    none = fa.Tensor.empty(device, (1, 2, 0, 64), dtype)
    how = dict(offset=350 - Sq, window=70, sinks=2)
    got = upload(device, c.q, dtype).flash_attention(*(upload(device, x, dtype) for x in (c.k, c.v)), c.scale, analytic=(True, 350 - Sq, 70), sinks=2,
                                                     prefix=(none, none))
    c.check(np.asarray(got.to_numpy(), np.float32), **how)


def test_many_rows(device):
    """More rows than a launch has in one dimension at a wavefront each: in the kernel that takes every call, and in a tiled one."""
    for D in (12, 16):
        B, H, Sq = 1 << 15, 4, 600
        n = B * H * Sq
        q = fa.Tensor.empty(device, (B, H, Sq, D), fa.F16)
        fa.check(fa.lib().fhip_memset(device.stream, ctypes.c_void_p(q.buffer.ptr), 0, q.buffer.nbytes))
        k = upload(device, np.ones((1, 1, 2, D)), fa.F16)
        v = upload(device, np.broadcast_to(np.asarray([1.0, 3.0])[None, None, :, None], (1, 1, 2, D)), fa.F16)
        whole = [fa.Tensor(t.buffer, fa.F16, (B, 1, 2, D), (0, *t.strides[1:])) for t in (k, v)]
        out = q.flash_attention(*whole, 0.5, prefix=(k, v))  # (scores of nothing: the mean of 1, 3, 1, 3)
        assert n * 64 > 1 << 32
        for at in (0, n - 1, (1 << 26) + 5):
            host = np.empty(D, np.float16)
            fa.check(fa.lib().fhip_memcpy_d2h(device.stream, host.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(out.buffer.ptr + at * D * 2), 2 * D))
            assert (host == 2.0).all(), (D, at)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Sq", [1, 40, 200])
@pytest.mark.parametrize("D", [64, 72, 256])
def test_broadcast_inputs(device, dtype, Sq, D):
    """Queries that heads share, keys that the batch or its heads share, one row of values for all keys."""
    B, H, Hkv, Skv, P = 2, 4, 2, 210, 90
    c = Call(device, dtype, B, H, Hkv, Sq, Skv, P, D, seed=16)
    c.q[:] = c.q[:, :1]
    c.k[:] = c.k[:1, :1]
    c.v[:] = c.v[:1, :, :1]
    c.pk[:] = c.pk[:1]
    c.pv[:] = c.pv[:, :1]

    def shared(x, *dims):
        """x with one element of memory along `dims`."""
        t = upload(device, x[tuple(slice(0, 1) if i in dims else slice(None) for i in range(4))], dtype)
        return fa.Tensor(t.buffer, dtype, x.shape, [0 if i in dims else s for i, s in enumerate(t.strides)])

    tensors = [shared(c.q, 1), shared(c.k, 0, 1), shared(c.v, 0, 2), shared(c.pk[None], 1), shared(c.pv[None], 2)]
    for how in (dict(offset=P + Skv - Sq), dict(offset=P + Skv - Sq, window=150, sinks=5)):
        c.check(c.run(tensors=tensors, **how), **how)
