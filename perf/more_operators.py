"""Attention whose keys come in two parts, as cases that can be timed and compared.

Two operators, reached through Tensor.flash_attention:

  sinks   a sliding window whose first tokens stay visible: a row at position p sees the keys j <= p with j + window > p or j < sinks
  prefix  a batch that shares a long prefix: keys and values of the prefix are held once, [1, kv_heads, prefix, head_dim], in front of
          every sequence's own, [batch, kv_heads, own, head_dim]; a window and sinks count positions from the prefix's first key

Each for one new token per sequence, a draft of a few, a chunk of a prompt, a whole prompt, in f32, f16 and bf16.
"""
import math
import random

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _case(kind, dtype, batch, heads, kv_heads, head_dim, rows, keys, prefix=0, window=0, sinks=0, ragged=False, name=None):
    """keys: what the cache of a sequence holds, the new rows among them (ragged: at most), without the prefix."""
    c = dict(kind=kind, dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, rows=rows, keys=keys, prefix=prefix,
             window=window, sinks=sinks, ragged=ragged)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one chat stream generating a token on a context of 4200 positions, in the reference's f32
        _case("sinks", "f32", 1, 32, 8, 128, 1, 4200, window=1024, sinks=4, name="sink_chat_step_f32"),
        # a serving batch generating one token per sequence, contexts of 2000 to 16384 tokens
        _case("sinks", "f16", 16, 32, 8, 128, 1, 16384, window=4096, sinks=16, ragged=True, name="sink_decode_ragged_f16"),
        # a draft of four tokens per sequence checked at key length 256, odd length
        _case("sinks", "bf16", 8, 16, 4, 256, 4, 4001, window=1024, sinks=5, name="sink_draft_d256_bf16"),
        # a prompt of 8192 tokens under half of it as window
        _case("sinks", "f16", 1, 32, 8, 128, 8192, 8192, window=4096, sinks=64, name="sink_prompt_f16"),
        # the next 512 tokens of four long prompts fed in chunks
        _case("sinks", "bf16", 4, 32, 8, 128, 512, 16896, window=4096, sinks=128, name="sink_chunk_bf16"),
        # a follow-up message on a long conversation in f32: odd sizes, heads that are not grouped, a head_dim that is no power of two
        _case("sinks", "f32", 1, 16, 16, 80, 129, 8003, window=2048, sinks=4, name="sink_turn_d80_f32"),
        # a few sequences of a small model that have just left a short system prompt
        _case("prefix", "f32", 4, 8, 4, 64, 1, 77, prefix=301, ragged=True, name="prefix_few_d64_f32"),
        # a serving batch behind a long instruction, answers of up to 1024 tokens so far
        _case("prefix", "f16", 32, 32, 8, 128, 1, 1024, prefix=8192, ragged=True, name="prefix_decode_f16"),
        # the same without grouped heads, one document asked 48 questions
        _case("prefix", "bf16", 48, 32, 32, 96, 1, 515, prefix=4096, ragged=True, name="prefix_decode_mha_d96_bf16"),
        # drafts of four tokens at key length 256
        _case("prefix", "f16", 16, 16, 4, 256, 4, 600, prefix=4001, ragged=True, name="prefix_draft_d256_f16"),
        # eight questions of 257 tokens each about one document, as they come in
        _case("prefix", "f16", 8, 32, 8, 128, 257, 257, prefix=8192, name="prefix_questions_f16"),
        # a batch in f32 whose model has a window and sinks: the sinks and part of the window lie in the prefix
        _case("prefix", "f32", 16, 32, 8, 128, 1, 1500, prefix=4096, window=4096, sinks=4, ragged=True, name="prefix_window_sinks_f32"),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm: odd ones as often as even ones."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind, dtype = rng.choice(["sinks", "prefix"]), rng.choice(["f32", "f16", "bf16"])
    heads, kv_heads = rng.choice([(32, 8), (16, 4), (16, 16), (8, 4), (32, 32)])
    head_dim = rng.choice([64, 80, 96, 128, 128, 256])
    if head_dim == 256 and heads == 32:
        heads, kv_heads = 16, 4
    shape = rng.choice(["token", "token", "draft", "prompt"])
    rows = 1 if shape == "token" else rng.randint(2, 8) if shape == "draft" else _between(rng, 9, 2000)
    sinks, window = _between(rng, 1, 128), _between(rng, 100, 5000)
    if kind == "sinks":
        if shape == "prompt":
            keys, batch = rows + rng.choice([0, _between(rng, 100, 12000)]), rng.choice([1, 1, 2])
            return _case(kind, dtype, batch, heads, kv_heads, head_dim, rows, keys, window=window, sinks=sinks)
        keys = _between(rng, 300, 16000)
        most = int(1.5e9 / (2 * kv_heads * keys * head_dim))
        batch = _between(rng, 1, max(1, min(32, most)))
        return _case(kind, dtype, batch, heads, kv_heads, head_dim, rows, keys, window=window, sinks=sinks, ragged=rng.random() < 0.5)
    prefix = _between(rng, 200, 12000)
    if shape == "prompt":
        rows = min(rows, 400)
        batch = _between(rng, 2, max(2, min(8, 1600 // rows)))
        keys, ragged = rows + rng.choice([0, _between(rng, 1, 1000)]), False
    else:
        batch = _between(rng, 2, 64)
        keys, ragged = rows + _between(rng, 1, 1500), rng.random() < 0.7
    if rng.random() < 0.7:
        window = sinks = 0
    return _case(kind, dtype, batch, heads, kv_heads, head_dim, rows, keys, prefix=prefix, window=window, sinks=sinks, ragged=ragged)


def _lengths(c, seed=0):
    """Keys of their own that the sequences of a batch hold, the new rows among them."""
    if not c["ragged"]:
        return [c["keys"]] * c["batch"]
    r = random.Random(c["batch"] * 100003 + c["keys"])
    low = min(c["keys"], max(c["rows"], c["keys"] // 8))
    got = [r.randint(low, c["keys"]) for _ in range(c["batch"])]
    random.Random(seed).shuffle(got)
    return got


# ---- the plain form --------------------------------------------------------------------------------------------------------------------


def _hidden(s):
    """[batch or 1, rows, prefix + keys]: what the rows of a sequence do not see."""
    c = s["case"]
    P, n = c["prefix"], c["rows"]
    key = torch.arange(P + c["keys"], device="cuda")
    length = s["lens_gpu"].view(-1, 1, 1) if c["ragged"] else torch.full((1, 1, 1), c["keys"], device="cuda")
    position = P + length - n + torch.arange(n, device="cuda").view(1, n, 1)
    hidden = key > position
    if c["window"]:
        hidden |= (key + c["window"] <= position) & (key >= c["sinks"])
    return hidden


def _plain(s):
    c = s["case"]
    B, H, Hkv, D, n, P, keys = (c[k] for k in ("batch", "heads", "kv_heads", "head_dim", "rows", "prefix", "keys"))
    G = H // Hkv
    q = s["q"].float()
    scores = torch.matmul(q.reshape(B, Hkv, G * n, D), s["k"].float().transpose(-1, -2).contiguous()).view(B, H, n, keys)
    if P:
        # every sequence's rows meet the prefix in one product
        folded = q.view(B, Hkv, G * n, D).transpose(0, 1).reshape(Hkv, B * G * n, D)
        front = torch.matmul(folded, s["pk"][0].float().transpose(-1, -2).contiguous())
        front = front.view(Hkv, B, G, n, P).transpose(0, 1).reshape(B, H, n, P)
        scores = torch.cat([front, scores], -1)
    scores = scores * s["scale"]
    scores.masked_fill_(_hidden(s).unsqueeze(1), -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores[..., P:].reshape(B, Hkv, G * n, keys), s["v"].float()).view(B, H, n, D)
    if P:
        folded = scores[..., :P].reshape(B, Hkv, G * n, P).transpose(0, 1).reshape(Hkv, B * G * n, P)
        front = torch.matmul(folded, s["pv"][0].float())
        out = out + front.view(Hkv, B, G, n, D).transpose(0, 1).reshape(B, H, n, D)
    return (out / total).transpose(1, 2).to(TORCH[c["dtype"]])


# ---- inputs ----------------------------------------------------------------------------------------------------------------------------


class _Memory:
    """Memory of a torch tensor as a buffer of the framework."""

    def __init__(self, device, tensor):
        self.device, self.tensor, self.ptr = device, tensor, tensor.data_ptr()


def _wrap(fa, device, tensor):
    return fa.Tensor(_Memory(device, tensor), {torch.float32: fa.F32, torch.float16: fa.F16, torch.bfloat16: fa.BF16}[tensor.dtype],
                     tuple(tensor.shape))


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, H, Hkv, D, n, P = (c[k] for k in ("batch", "heads", "kv_heads", "head_dim", "rows", "prefix"))

    def normal(*shape):
        return torch.empty(shape, device="cuda").normal_(0.0, 1.0, generator=gen)

    s = dict(case=c, scale=D ** -0.5)
    # queries lean towards one direction of their KV head, and the first keys lie along it: they draw weight, as first tokens do
    lean = normal(1, Hkv, 1, D)
    k, v, q = normal(B, Hkv, c["keys"], D), normal(B, Hkv, c["keys"], D), normal(B, H, n, D)
    if P:
        pk, pv = normal(1, Hkv, P, D), normal(1, Hkv, P, D)
    first = pk if P else k
    first[:, :, :max(1, c["sinks"])] += 0.3 * lean
    q += lean.repeat_interleave(H // Hkv, 1)
    for name, x in (("q", q), ("k", k), ("v", v)) + ((("pk", pk), ("pv", pv)) if P else ()):
        s[name] = x.to(TORCH[c["dtype"]])
    # as the projection behind attention reads it: [batch, rows, heads, head_dim]
    s["out"] = torch.empty(B, n, H, D, dtype=TORCH[c["dtype"]], device="cuda")
    s["lens"] = _lengths(c, seed)
    s["lens_gpu"] = torch.tensor(s["lens"], device="cuda") if c["ragged"] else None
    if own:
        _bind(s)
    torch.cuda.synchronize()
    return s


def _bind(s):
    """The framework's handles of a state's memory."""
    import floneum_amd as fa
    c, dev = s["case"], fa.Device.default()
    s["fa_q"], s["fa_k"], s["fa_v"] = (_wrap(fa, dev, s[x]) for x in "qkv")
    s["fa_prefix"] = (_wrap(fa, dev, s["pk"]), _wrap(fa, dev, s["pv"])) if c["prefix"] else None
    s["fa_out"] = _wrap(fa, dev, s["out"]).transpose(1, 2)
    s["fa_lens"] = s["fa_positions"] = None
    s["analytic"] = (True, c["prefix"] + (0 if c["ragged"] else c["keys"] - c["rows"]), c["window"])
    if c["ragged"]:
        s["fa_lens"] = fa.IntTensor(dev, np.asarray(s["lens"], np.int32))
        s["fa_positions"] = fa.IntTensor(dev, np.asarray(s["lens"], np.int32) - c["rows"])


def run(s):
    if not own:
        return _plain(s)
    s["fa_q"].flash_attention(s["fa_k"], s["fa_v"], s["scale"], analytic=s["analytic"], sinks=s["case"]["sinks"], prefix=s["fa_prefix"],
                              kv_lens=s["fa_lens"], q_positions=s["fa_positions"], out=s["fa_out"])
    return s["out"]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------------------


def work(case):
    c = case
    D, n, P, window = c["head_dim"], c["rows"], c["prefix"], c["window"]
    pairs = own_seen = 0
    front = np.zeros(P, bool)
    for length in _lengths(c):
        position = np.arange(P + length - n, P + length, dtype=np.int64)
        low = np.maximum(position - window + 1, 0) if window else 0 * position
        sinks = np.minimum(c["sinks"], low)  # those below the row's window
        pairs += int(np.sum(position + 1 - low + sinks))
        most, least = int(sinks.max()), int(low.min())
        front[least:] = True
        front[:most] = True
        own_seen += P + length - max(P, least) + max(0, min(most, least) - P)
    b = BYTES[c["dtype"]]
    return {"bytes": 2 * b * D * (c["batch"] * c["heads"] * n + c["kv_heads"] * (int(front.sum()) + own_seen)), "flops": 4 * D * c["heads"] * pairs}


# ---- the same from the definition, in 64 bits ------------------------------------------------------------------------------------------


def exact(case, seed):
    c, s = case, prepare(case, seed)
    f64 = torch.float64
    group, P = c["heads"] // c["kv_heads"], c["prefix"]
    out = torch.empty(s["out"].shape, dtype=f64, device="cuda")
    for b in range(c["batch"]):
        length = s["lens"][b]
        at = torch.arange(P + length - c["rows"], P + length, device="cuda")[:, None] - torch.arange(P + length, device="cuda")[None, :]
        seen = at >= 0
        if c["window"]:
            seen &= (at < c["window"]) | (torch.arange(P + length, device="cuda") < c["sinks"])[None, :]
        for g in range(c["kv_heads"]):
            k, v = (torch.cat([s["p" + x][0, g], s[x][b, g, :length]]) if P else s[x][b, g, :length] for x in "kv")
            k, v = k.to(f64), v.to(f64)
            for h in range(g * group, (g + 1) * group):
                x = torch.where(seen, (s["q"][b, h].to(f64) @ k.T) * s["scale"], -math.inf)
                out[b, :, h] = torch.softmax(x, -1) @ v
    return out
