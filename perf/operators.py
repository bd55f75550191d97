"""The work that users of this framework have its 8-bit key / value cache do, as cases that can be timed and compared.

Three operators, each through the package's public entry points:

  append  the step before attention: q and the new keys rotated (and normalised first, in models that have such norms), new
          keys and values into the 8-bit cache, one scale per block of tokens and head; the rows that were written are read back,
          with the earlier rows of the blocks that they fell into
  read    a stretch of the cache read back as ordinary numbers
  attend  attention over the 8-bit cache: one new token per sequence, a draft of a few, a chunk of a prompt, a whole prompt

A cache holds [batch, kv_heads, rows, head_dim] codes of 8 bits ("int8": -127..127, "e4m3": the 8-bit float with 4 exponent and 3
mantissa bits) and an f32 scale per (batch, kv head, block of tokens).  A block's scale is the largest magnitude of its rows over the largest
code, in f32; a code is the nearest one of value / scale, ties to even.  Rows that join a block raise its scale if they have to, and the
rows that were there are then coded again from what they read back as.
"""
import math
import random

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
LARGEST = {"int8": 127.0, "e4m3": 448.0}
SMALLEST_SCALE = 2.0 ** -100


def _append(dtype, batch, heads, kv_heads, head_dim, rows, fmt, block, norm=False, lens=0, back="f32", name=None):
    c = dict(kind="append", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rows=rows, format=fmt,
             block=block, norm=norm, lens=lens, back=back)
    return c if name is None else dict(c, name=name)


def _read(back, batch, kv_heads, head_dim, rows, fmt, block, name=None):
    c = dict(kind="read", back=back, batch=batch, kv_heads=kv_heads, head_dim=head_dim, rows=rows, format=fmt, block=block)
    return c if name is None else dict(c, name=name)


def _attend(dtype, batch, heads, kv_heads, head_dim, rows, keys, fmt, block, causal=False, window=0, ragged=False, name=None):
    c = dict(kind="attend", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rows=rows, keys=keys, format=fmt,
             block=block, causal=causal, window=window, ragged=ragged)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # the new token of 16 streams whose caches hold different numbers of tokens
        _append("f16", 16, 32, 8, 128, 1, "int8", 1, lens=4000, name="append_token_int8"),
        # the same with q / k norms and a key length of 256, into blocks of 32 tokens that are partly filled
        _append("bf16", 64, 16, 4, 256, 1, "e4m3", 32, norm=True, lens=4000, back="bf16", name="append_token_blocks_e4m3"),
        # a prompt of 8192 tokens on its way into the cache
        _append("f16", 1, 32, 8, 128, 8192, "int8", 1, back="f16", name="append_prompt_int8"),
        # a short conversation read back, odd length
        _read("f32", 1, 8, 64, 301, "int8", 1, name="read_chat_int8"),
        # a serving batch's layer read back
        _read("bf16", 16, 8, 128, 4096, "e4m3", 64, name="read_batch_e4m3"),
        # one chat stream generating a token on a context of 4096 positions, queries in the reference's f32
        _attend("f32", 1, 32, 8, 128, 1, 4096, "int8", 1, name="chat_step_int8_f32"),
        # a serving batch generating one token per sequence
        _attend("f16", 16, 32, 8, 128, 1, 4096, "int8", 1, name="decode_batch_int8_f16"),
        # a ragged serving batch without grouped heads: 128 to 16384 cached keys per sequence
        _attend("f16", 16, 32, 32, 96, 1, 16384, "e4m3", 32, ragged=True, name="decode_ragged_e4m3_f16"),
        # a draft of four tokens per sequence checked at key length 256, odd length
        _attend("bf16", 8, 16, 4, 256, 4, 4001, "int8", 64, causal=True, name="draft_d256_int8_bf16"),
        # a prompt of 8192 tokens
        _attend("f16", 1, 32, 8, 128, 8192, 8192, "int8", 1, causal=True, name="prompt_int8_f16"),
        # the next 512 tokens of four prompts fed in chunks under a window of 4096 keys
        _attend("bf16", 4, 32, 8, 128, 512, 4607, "e4m3", 16, causal=True, window=4096, name="window_chunk_e4m3_bf16"),
        # a follow-up message on a long conversation, queries in f32: odd sizes, few rows on many keys
        _attend("f32", 1, 32, 8, 128, 129, 8003, "int8", 1, causal=True, name="chat_turn_int8_f32"),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm: odd ones as often as even ones."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "read", "attend", "attend", "attend", "attend"])
    dtype, fmt, block = rng.choice(["f32", "f16", "bf16"]), rng.choice(["int8", "e4m3"]), rng.choice([1, 1, 8, 16, 32, 64])
    heads, kv_heads = rng.choice([(32, 8), (16, 4), (16, 16), (8, 4), (32, 32)])
    head_dim = rng.choice([64, 80, 96, 128, 128, 256])
    if kind == "append":
        rows = rng.choice([1, 1, _between(rng, 2, 2000)])
        batch = _between(rng, 1, 64 if rows == 1 else 4)
        norm = dtype != "f32" and rng.random() < 0.4
        back = dtype if norm else rng.choice(["f32", "f16", "bf16"])
        return _append(dtype, batch, heads, kv_heads, head_dim, rows, fmt, block, norm, _between(rng, 1, 8000), back)
    if kind == "read":
        rows = _between(rng, 1, 16000)
        return _read(rng.choice(["f32", "f16", "bf16"]), _between(rng, 1, max(1, 60000 // rows)), kv_heads, head_dim, rows, fmt, block)
    shape = rng.choice(["token", "token", "draft", "prompt", "chunk", "turn"])
    if shape in ("token", "draft"):
        rows = 1 if shape == "token" else rng.randint(2, 8)
        keys = _between(rng, 300, 16000)
        most = int(1.5e9 / (2 * kv_heads * keys * head_dim))  # 1.5 GB of cache at most
        ragged = rng.random() < 0.3
        return _attend(dtype, _between(rng, 1, max(1, min(32, most))), heads, kv_heads, head_dim, rows, keys, fmt, block,
                       causal=rows > 1, window=rng.choice([0, 0, 1024]), ragged=ragged)
    if head_dim == 256 and heads == 32:
        heads, kv_heads = 16, 4
    if shape == "prompt":
        rows = keys = _between(rng, 100, 4000)
        return _attend(dtype, 1, heads, kv_heads, head_dim, rows, keys, fmt, block, causal=True)
    if shape == "chunk":
        rows = _between(rng, 100, 1000)
        return _attend(dtype, rng.choice([1, 2]), heads, kv_heads, head_dim, rows, rows + _between(rng, 1000, 7000), fmt, block, causal=True,
                       window=4096)
    rows = _between(rng, 9, 300)
    return _attend(dtype, 1, heads, kv_heads, head_dim, rows, rows + _between(rng, 1000, 16000), fmt, block, causal=True)


def _lengths(c, seed=0):
    """Tokens that the sequences of a batch hold, spread evenly over what such a batch has."""
    r = random.Random(c["batch"] * 100003 + (c["lens"] if c["kind"] == "append" else c["keys"]))
    if c["kind"] == "append":
        got = [r.randint(min(c["lens"], c["lens"] // 8), c["lens"]) for _ in range(c["batch"])]
    else:
        low = min(c["keys"], max(128, c["rows"]))
        got = [r.randint(low, c["keys"]) for _ in range(c["batch"])]
    random.Random(seed).shuffle(got)
    return got


def _capacity(c):
    """Rows that an append case's cache has room for: whole blocks."""
    return (c["lens"] + c["rows"] + c["block"] - 1) // c["block"] * c["block"]


# ---- the plain form --------------------------------------------------------------------------------------------------------------------


def _nearest(y, fmt):
    """The codes' values nearest to y (64 bits), ties to even."""
    if fmt == "int8":
        return y.round().clamp(-127.0, 127.0)
    exponent = torch.frexp(y)[1].clamp(min=-5) - 1  # of the leading bit; below 2^-6 the steps stay as they are
    step = torch.ldexp(torch.ones_like(y), exponent - 3)
    return ((y / step).round() * step).clamp(-448.0, 448.0)


def _stored(values, fmt):
    return values.to(torch.int8 if fmt == "int8" else torch.float8_e4m3fn)


def _scales(x, fmt, block, before=None):
    """f32 scales [..., blocks] of x [..., rows, head_dim] (whole blocks), at least `before`."""
    b = x.abs().amax(-1).unflatten(-1, (-1, block)).amax(-1) / LARGEST[fmt]
    b = torch.where(torch.isfinite(b), b, torch.full_like(b, math.nan)).clamp(min=SMALLEST_SCALE)
    return b if before is None else torch.maximum(b, before)


def _spread(scales, block):
    return scales.repeat_interleave(block, -1).unsqueeze(-1)


def _values(codes, scales, block, rows):
    """What rows 0.. of a cache stand for, in f32."""
    return codes[..., :rows, :].float() * _spread(scales, block)[..., :rows, :]


def _normed(x, weight, eps, dtype):
    """Root-mean-square norm of x's rows, rounded to their type."""
    x32 = x.float()
    mean = x.double().square().mean(-1, keepdim=True).float()
    return (x32 / torch.sqrt(mean + eps) * weight.float()).to(TORCH[dtype])


def _rotated(x, cos, sin):
    """Pairs (i, i + head_dim / 2) of x turned by the angles of its rows' positions, in f32."""
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    c = s["case"]
    n, block, fmt = c["rows"], c["block"], c["format"]
    at = s["lens_gpu"][:, None] + torch.arange(n, device="cuda")[None, :]  # [batch, rows]
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q, k, v = s["q"].transpose(1, 2), s["k"].transpose(1, 2), s["v"].transpose(1, 2)
    if c["norm"]:
        q, k = _normed(q, s["q_weight"], s["eps"], c["dtype"]), _normed(k, s["k_weight"], s["eps"], c["dtype"])
    q_out = _rotated(q, cos, sin).to(TORCH[c["dtype"]])
    out = [q_out]
    first = s["lens_gpu"] // block * block
    span = (n + 2 * (block - 1)) // block * block  # whole blocks, enough for any place in the first one
    rows = first[:, None] + torch.arange(span, device="cuda")[None, :]
    inside = (rows < s["k_codes"].shape[2])
    taken = rows.clamp(max=s["k_codes"].shape[2] - 1)
    batch = torch.arange(c["batch"], device="cuda")[:, None]
    new = (rows >= s["lens_gpu"][:, None]) & (rows < s["lens_gpu"][:, None] + n)
    index = (rows - s["lens_gpu"][:, None]).clamp(0, n - 1)
    started = (s["lens_gpu"] % block != 0)[:, None, None]
    for x, codes, scales in ((_rotated(k, cos, sin), s["k_codes"], s["k_scales"]), (v.float(), s["v_codes"], s["v_scales"])):
        old_scales = scales[batch, :, taken[:, ::block] // block].transpose(1, 2)
        old = codes.view(torch.int8)[batch, :, taken].view(codes.dtype).transpose(1, 2).float() * _spread(old_scales, block)
        x = x.transpose(1, 2)[batch, index].transpose(1, 2)
        there = (rows < s["lens_gpu"][:, None])[:, None, :, None]
        fresh = torch.where(new[:, None, :, None], x, torch.zeros_like(x))
        before = torch.zeros_like(old_scales)
        before[:, :, :1] = torch.where(started, old_scales[:, :, :1], before[:, :, :1])
        now = _scales(fresh, fmt, block, before)
        value = torch.where(there, old, fresh)
        value = _nearest(value.double() / _spread(now, block).double(), fmt).float() * _spread(now, block)
        value = torch.where((there | new[:, None, :, None]) & inside[:, None, :, None], value, torch.zeros_like(value))
        out.append(value[:, :, :s["read_rows"]].to(TORCH[c["back"]]))
    return out


def _plain_attend(s):
    c = s["case"]
    B, H, Hkv, D, n, keys = (c[k] for k in ("batch", "heads", "kv_heads", "head_dim", "rows", "keys"))
    k = _values(s["k_codes"], s["k_scales"], c["block"], keys)
    v = _values(s["v_codes"], s["v_scales"], c["block"], keys)
    scores = torch.matmul(s["q"].float().reshape(B, Hkv, H // Hkv * n, D), k.transpose(-1, -2).contiguous()) * s["scale"]
    scores = scores.view(B, H, n, keys)
    if c["causal"] or c["ragged"]:
        key, row = torch.arange(keys, device="cuda"), torch.arange(n, device="cuda")[:, None]
        length = s["lens_gpu"][:, None, None] if c["ragged"] else keys
        position = length - n + row
        hidden = (key > position) if c["causal"] else (key >= length)
        if c["causal"] and c["window"]:
            hidden = hidden | (key + c["window"] <= position)
        scores.masked_fill_(hidden.unsqueeze(1) if c["ragged"] else hidden, -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(B, Hkv, H // Hkv * n, keys), v).view(B, H, n, D) / total
    return out.transpose(1, 2).to(TORCH[c["dtype"]])


# ---- inputs ----------------------------------------------------------------------------------------------------------------------------


class _Memory:
    """Memory of a torch tensor as a buffer of the framework."""

    def __init__(self, device, tensor):
        self.device, self.tensor, self.ptr = device, tensor, tensor.data_ptr()


def _wrap(fa, device, tensor):
    return fa.Tensor(_Memory(device, tensor), {torch.float32: fa.F32, torch.float16: fa.F16, torch.bfloat16: fa.BF16}[tensor.dtype],
                     tuple(tensor.shape))


def _wrap8(fa, device, codes, scales, case):
    fmt = fa.Q8Format.INT8 if case["format"] == "int8" else fa.Q8Format.E4M3
    return fa.Q8Tensor(_Memory(device, codes), _Memory(device, scales), tuple(codes.shape), fmt, case["block"])


def _coded(x, fmt, block):
    """Codes and scales of x [batch, kv_heads, rows, head_dim], a part of the batch at a time: (codes of whole blocks, scales)."""
    rows = x.shape[2]
    whole = (rows + block - 1) // block * block
    codes = torch.zeros(x.shape[0], x.shape[1], whole, x.shape[3], dtype=torch.int8 if fmt == "int8" else torch.float8_e4m3fn, device="cuda")
    scales = torch.zeros(x.shape[0], x.shape[1], whole // block, device="cuda")
    for b in range(x.shape[0]):
        padded = torch.nn.functional.pad(x[b].float(), (0, 0, 0, whole - rows))
        scales[b] = _scales(padded, fmt, block)
        codes[b] = _stored(_nearest((padded / _spread(scales[b], block)).double(), fmt).float(), fmt)
    return codes, scales


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, Hkv, D, block, fmt = (c[k] for k in ("batch", "kv_heads", "head_dim", "block", "format"))

    def normal(*shape, dtype="f32", std=1.0, mean=0.0):
        return torch.empty(shape, device="cuda").normal_(mean, std, generator=gen).to(TORCH[dtype])

    s = dict(case=c)
    kept = c["lens"] if c["kind"] == "append" else c["rows"] if c["kind"] == "read" else c["keys"]
    for side in ("k", "v")[: 1 if c["kind"] == "read" else 2]:
        s[side + "_codes"], s[side + "_scales"] = _coded(normal(B, Hkv, kept, D, dtype="f16"), fmt, block)
    if c["kind"] == "append":
        n, room = c["rows"], _capacity(c)
        s["lens"] = _lengths(c, seed)
        s["lens_gpu"] = torch.tensor(s["lens"], device="cuda")
        behind = torch.arange(room, device="cuda")[None, :] >= s["lens_gpu"][:, None]  # rows that are not written yet
        for side in "kv":
            codes = torch.zeros(B, Hkv, room, D, dtype=s[side + "_codes"].dtype, device="cuda")
            codes[:, :, :min(room, s[side + "_codes"].shape[2])] = s[side + "_codes"][:, :, :room]
            codes.view(torch.int8).masked_fill_(behind[:, None, :, None], 0)
            scales = torch.zeros(B, Hkv, room // block, device="cuda")
            scales[:, :, :s[side + "_scales"].shape[2]] = s[side + "_scales"]
            s[side + "_codes"], s[side + "_scales"] = codes, scales
        # projections as a model holds them, [batch, rows, heads, head_dim]
        s["q"] = normal(B, n, c["heads"], D, dtype=c["dtype"])
        s["k"], s["v"] = normal(B, n, Hkv, D, dtype=c["dtype"], std=1.1), normal(B, n, Hkv, D, dtype=c["dtype"], std=1.1)
        s["q_weight"], s["k_weight"], s["eps"] = normal(D, mean=1.0, std=0.2), normal(D, mean=1.0, std=0.2), 1e-6
        angles = torch.arange(room + 1, device="cuda").double()[:, None] * 10000.0 ** (-torch.arange(0, D, 2, device="cuda").double() / D)
        s["cos"], s["sin"] = angles.cos().float(), angles.sin().float()
        s["read_rows"] = n + block - 1
        s["out"] = [torch.zeros(B, c["heads"], n, D, dtype=TORCH[c["dtype"]], device="cuda")]
        s["out"] += [torch.zeros(B, Hkv, s["read_rows"], D, dtype=TORCH[c["back"]], device="cuda") for _ in range(2)]
    elif c["kind"] == "read":
        s["out"] = torch.empty(B, Hkv, c["rows"], D, dtype=TORCH[c["back"]], device="cuda")
    else:
        s["scale"] = D ** -0.5
        s["q"] = normal(B, c["heads"], c["rows"], D, dtype=c["dtype"])
        # as the projection behind attention reads it: [batch, rows, heads, head_dim]
        s["out"] = torch.empty(B, c["rows"], c["heads"], D, dtype=TORCH[c["dtype"]], device="cuda")
        s["lens"] = _lengths(c, seed) if c["ragged"] else None
        s["lens_gpu"] = torch.tensor(s["lens"], device="cuda") if c["ragged"] else None
    if own:
        _bind(s)
    torch.cuda.synchronize()
    return s


def _bind(s):
    """The framework's handles of a state's memory."""
    import floneum_amd as fa
    c, dev = s["case"], fa.Device.default()
    s["k8"] = _wrap8(fa, dev, s["k_codes"], s["k_scales"], c)
    if c["kind"] == "read":
        s["fa_out"] = _wrap(fa, dev, s["out"])
        return
    s["v8"] = _wrap8(fa, dev, s["v_codes"], s["v_scales"], c)
    s["fa_lens"] = None if s["lens"] is None else fa.IntTensor(dev, np.asarray(s["lens"], np.int32))
    if c["kind"] == "append":
        s["fa_q"], s["fa_k"], s["fa_v"] = (_wrap(fa, dev, s[x]).transpose(1, 2) for x in "qkv")
        s["fa_out"] = [_wrap(fa, dev, x) for x in s["out"]]
        s["rope"] = fa.RopeCache.from_parts(s["cos"].cpu().numpy(), s["sin"].cpu().numpy(), dev)
        s["q_norm"] = s["k_norm"] = None
        if c["norm"]:
            s["q_norm"], s["k_norm"] = (fa.RmsNorm(s[x].cpu().numpy(), None, s["eps"], fa.F32, dev) for x in ("q_weight", "k_weight"))
        s["fa_first"] = fa.IntTensor(dev, np.asarray(s["lens"], np.int32) // c["block"] * c["block"])
        return
    s["fa_q"], s["fa_out"] = _wrap(fa, dev, s["q"]), _wrap(fa, dev, s["out"]).transpose(1, 2)
    s["analytic"], s["positions"] = None, None
    if c["causal"]:
        s["analytic"] = (True, 0 if c["ragged"] else c["keys"] - c["rows"], c["window"])
        if c["ragged"]:
            s["positions"] = fa.IntTensor(dev, np.asarray(s["lens"], np.int32) - c["rows"])


def run(s):
    kind = s["case"]["kind"]
    if own:
        if kind == "append":
            s["k8"].append(s["v8"], s["fa_k"], s["fa_v"], lens=s["fa_lens"], rope=s["rope"], k_norm=s["k_norm"], q=s["fa_q"],
                           q_norm=s["q_norm"], q_out=s["fa_out"][0])
            s["k8"].dequantize(out=s["fa_out"][1], lens=s["fa_first"])
            s["v8"].dequantize(out=s["fa_out"][2], lens=s["fa_first"])
        elif kind == "read":
            s["k8"].narrow(2, 0, s["case"]["rows"]).dequantize(out=s["fa_out"])
        else:
            keys = s["case"]["keys"]
            s["fa_q"].flash_attention(s["k8"].narrow(2, 0, keys), s["v8"].narrow(2, 0, keys), s["scale"], analytic=s["analytic"],
                                      kv_lens=s["fa_lens"], q_positions=s["positions"], out=s["fa_out"])
        return s["out"]
    if kind == "append":
        return _plain_append(s)
    if kind == "read":
        return _values(s["k_codes"], s["k_scales"], s["case"]["block"], s["case"]["rows"]).to(TORCH[s["case"]["back"]])
    return _plain_attend(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------------


def _seen(c):
    """(keys that some row of a sequence sees, pairs of query row and key that count), summed over the batch."""
    seen = pairs = 0
    for length in _lengths(c) if c["ragged"] else [c["keys"]] * c["batch"]:
        if not c["causal"]:
            seen, pairs = seen + length, pairs + c["rows"] * length
            continue
        position = np.arange(length - c["rows"], length, dtype=np.int64)
        low = np.maximum(position - c["window"] + 1, 0) if c["window"] else 0 * position
        seen, pairs = seen + length - int(low[0]), pairs + int(np.sum(position + 1 - low))
    return seen, pairs


def work(case):
    c = case
    B, Hkv, D, block = (c[k] for k in ("batch", "kv_heads", "head_dim", "block"))
    row = D + 4 / block  # a cached row of one head
    if c["kind"] == "read":
        return {"bytes": B * Hkv * c["rows"] * (row + D * BYTES[c["back"]]), "flops": B * Hkv * c["rows"] * D}
    e, H, n = BYTES[c["dtype"]], c["heads"], c["rows"]
    if c["kind"] == "append":
        earlier = sum(length % block for length in _lengths(c))
        written = B * n + earlier  # rows of the blocks that the new ones fall into
        b = e * B * n * D * (2 * H + 2 * Hkv) + 2 * Hkv * row * (2 * written + earlier) + 2 * Hkv * D * BYTES[c["back"]] * B * (n + block - 1)
        return {"bytes": b + 4 * D * (B * n + 2 * c["norm"]), "flops": B * n * D * (3 * (H + Hkv) + 4 * Hkv) + 4 * Hkv * D * written}
    seen, pairs = _seen(c)
    return {"bytes": 2 * e * B * H * n * D + 2 * Hkv * seen * row, "flops": 4 * D * H * pairs}


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------------------------


def _exact_code(y, fmt):
    if fmt == "int8":
        return torch.round(y)
    power = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    power = torch.where(y.abs() >= torch.exp2(power + 1), power + 1, power)
    return torch.round(y * torch.exp2(3 - power)) * torch.exp2(power - 3)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    f64 = torch.float64
    B, Hkv, D, block, fmt = (c[k] for k in ("batch", "kv_heads", "head_dim", "block", "format"))

    def rows_of(side, b, lo, hi):
        index = torch.arange(lo, hi, device="cuda") // block
        return s[side + "_codes"][b, :, lo:hi].to(f64) * s[side + "_scales"][b][:, index, None].to(f64)

    if c["kind"] == "read":
        return torch.stack([rows_of("k", b, 0, c["rows"]) for b in range(B)])
    if c["kind"] == "attend":
        H, n, group = c["heads"], c["rows"], c["heads"] // Hkv
        out = torch.empty(B, n, H, D, dtype=f64, device="cuda")
        for b in range(B):
            length = s["lens"][b] if c["ragged"] else c["keys"]
            k, v = rows_of("k", b, 0, length), rows_of("v", b, 0, length)
            where = torch.arange(length - n, length, device="cuda")[:, None] - torch.arange(length, device="cuda")[None, :]
            for h in range(H):
                x = (s["q"][b, h].to(f64) @ k[h // group].T) * s["scale"]
                if c["causal"]:
                    x[where < 0] = -math.inf
                    if c["window"]:
                        x[where >= c["window"]] = -math.inf
                out[b, :, h] = torch.softmax(x, -1) @ v[h // group]
        return out
    n, half = c["rows"], D // 2
    outs = [torch.zeros(x.shape, dtype=f64, device="cuda") for x in s["out"]]
    for b in range(B):
        length = s["lens"][b]
        cos, sin = (s[x][length:length + n].to(f64)[:, None, :] for x in ("cos", "sin"))
        turned = {}
        for side in "qkv":
            x = s[side][b].to(f64)  # [rows, heads, head_dim]
            if side != "v":
                if c["norm"]:
                    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * s[side + "_weight"].to(f64)
                    x = x.to(TORCH[c["dtype"]]).to(f64)
                lo, hi = x[..., :half], x[..., half:]
                # the rotation is defined in f32: each product and each sum is rounded to it
                products = [(u * w).float().to(f64) for u, w in ((lo, cos), (-hi, sin), (hi, cos), (lo, sin))]
                x = torch.cat([products[0] + products[1], products[2] + products[3]], -1).float().to(f64)
            turned[side] = x.transpose(0, 1)
        outs[0][b] = turned["q"]
        first = length // block * block
        for at, side in ((1, "k"), (2, "v")):
            rows = torch.cat([rows_of(side, b, first, length), turned[side]], 1)  # from the start of the first block on
            for lo in range(0, rows.shape[1], block) if block > 1 else [0]:
                part = rows[:, lo:lo + block] if block > 1 else rows
                fresh = part[:, max(0, length - first - lo):] if block > 1 else part
                top = fresh.abs().amax((1, 2) if block > 1 else 2, keepdim=True) / LARGEST[fmt]
                top = top.float().to(f64).clamp(min=SMALLEST_SCALE)
                if block > 1 and length > first + lo:
                    top = torch.maximum(top, s[side + "_scales"][b][:, (first + lo) // block, None, None].to(f64))
                coded = _exact_code(part / top, fmt).clamp(-LARGEST[fmt], LARGEST[fmt]) * top
                outs[at][b][:, lo:lo + part.shape[1]] = coded[:, :max(0, outs[at].shape[2] - lo)]
    return outs
