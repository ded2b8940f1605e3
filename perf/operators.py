"""The operators of causal models that the library offers beside its encoder, each as one call: attention
over packed prompts and cached keys, attention of a batch over a shared prefix, and products of few rows
with 4-bit weights.

listed() names the cases, draw() gives others of the same ranges, prepare() makes a case's inputs on the
GPU, run() is one pass through an operator: the library's entries where `own` is set, else the plain torch
form in 32 bits. exact() states the same results in float64."""
import math
import os
import random
import sys
import zlib

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
GGUF_TYPES = {"f32": 0, "f16": 1, "q4_0": 2, "q4_1": 3, "bf16": 30}
BLOCK_BYTES = {"q4_0": 18, "q4_1": 20}
# Query heads, KV heads, head dim: the two text encoders' layers (window 512 and 1024 on the sliding
# ones), then the usual grouped, ungrouped and narrow layouts.
HEADS = [(3, 1, 256), (4, 2, 256), (4, 1, 512), (2, 1, 128), (32, 8, 128), (16, 16, 64), (12, 4, 64)]


def listed():
    return [
        # A search query read by a causal encoder: one short text, all latency.
        dict(name="query", kind="causal", type="f16", sequences=1, low=12, high=12, past_low=0, past_high=0,
             heads=3, kv_heads=1, head_dim=256, window=0, fused=False),
        # A ragged pack of passages on a sliding-window layer, q, k and v where the fused projection left them.
        dict(name="passages", kind="causal", type="bf16", sequences=9, low=130, high=997, past_low=0, past_high=0,
             heads=3, kv_heads=1, head_dim=256, window=512, fused=True),
        # A book chapter as one prompt, grouped heads.
        dict(name="chapter", kind="causal", type="f16", sequences=1, low=16384, high=16384, past_low=0, past_high=0,
             heads=32, kv_heads=8, head_dim=128, window=0, fused=False),
        # Documents read in chunks: 512 more tokens of each over the keys cached so far.
        dict(name="chunks", kind="causal", type="bf16", sequences=4, low=512, high=512, past_low=2000, past_high=9000,
             heads=16, kv_heads=16, head_dim=64, window=0, fused=False),
        # A serving step: one token for each of 48 texts over caches of different lengths.
        dict(name="steps", kind="causal", type="f16", sequences=48, low=1, high=1, past_low=100, past_high=8000,
             heads=32, kv_heads=8, head_dim=128, window=0, fused=False),
        # One text's next token after a task instruction, on the reference architecture's global layers.
        dict(name="instruction", kind="prefix", type="f16", prefix=300, sequences=1, low=1, high=1, past_low=8,
             past_high=8, heads=4, kv_heads=1, head_dim=512, window=0),
        # Candidates scored against one document: 64 texts, the next token of each.
        dict(name="candidates", kind="prefix", type="bf16", prefix=4096, sequences=64, low=1, high=1, past_low=0,
             past_high=200, heads=32, kv_heads=8, head_dim=128, window=0),
        # Many short texts embedded in the context of one long document.
        dict(name="contextual", kind="prefix", type="f16", prefix=8192, sequences=128, low=8, high=64, past_low=0,
             past_high=0, heads=3, kv_heads=1, head_dim=256, window=0),
        # The feed-forward's gate and up for one token of the encoder's width.
        dict(name="geglu_token", kind="q4", weights="q4_0", rows=1, width=768, features=1152, x="f16", y="f16",
             geglu=True),
        # One token through a large projection.
        dict(name="projection_token", kind="q4", weights="q4_0", rows=1, width=8192, features=8192, x="bf16", y="f32",
             geglu=False),
        # A dozen tokens through a wide feed-forward's gate and up.
        dict(name="geglu_dozen", kind="q4", weights="q4_1", rows=12, width=4096, features=11264, x="f16", y="f16",
             geglu=True),
        # A few texts' tokens through a head of an odd number of outputs.
        dict(name="projection_rows", kind="q4", weights="q4_1", rows=37, width=2048, features=1001, x="bf16", y="bf16",
             geglu=False),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["causal", "causal", "prefix", "q4"])
    if kind == "q4":
        geglu = rng.random() < 0.4
        return dict(kind=kind, weights=rng.choice(["q4_0", "q4_1"]), rows=rng.choice([1, 1, spread(2, 64)]),
                    width=32 * spread(8, 256), features=spread(64, 8192 if geglu else 12000),
                    x=rng.choice(["f16", "bf16"]), y=rng.choice(["f16", "bf16", "f32"]), geglu=geglu)
    heads, kv_heads, head_dim = rng.choice(HEADS)
    case = dict(kind=kind, type=rng.choice(["f16", "bf16"]))
    window = rng.choice([0, 0, 0, 512, 1024, spread(1, 4096)])
    if kind == "prefix":
        case.update(prefix=spread(16, 16384), sequences=spread(1, 256))
        # tokens of each text: one, or a short text's
        high = rng.choice([1, 1, min(spread(2, 128), max(1, 4096 // case["sequences"]))])
        past = rng.choice([0, spread(1, 512)])
        case.update(low=max(1, high // 4), high=high, past_low=past // 8, past_high=past)
    else:
        form = rng.choice(["prompt", "prompt", "chunk", "token"])
        if form == "prompt":
            high = spread(1, 8192)
            case.update(sequences=min(spread(1, 64), max(1, 16384 // high)), low=max(1, high // 8), high=high,
                        past_low=0, past_high=0)
        else:
            past = spread(16, 32768)
            high = 1 if form == "token" else spread(2, 512)
            case.update(sequences=min(spread(1, 128), max(1, 131072 // past)), low=max(1, high // 2), high=high,
                        past_low=past // 8, past_high=past)
    case.update(heads=heads, kv_heads=kv_heads, head_dim=head_dim, window=window)
    if kind == "causal":
        case["fused"] = case["past_high"] == 0 and rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------- inputs


def sequences(case):
    """(q_start, q_len, kv_start, kv_len) of each text: fixed by the case, the same for every seed. Queries
    are packed back to back; the keys of a cached text lie in a slot of their own with some rows to spare."""
    rng = random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    out, q, kv = [], 0, 0
    for _ in range(case["sequences"]):
        n = rng.randint(case["low"], case["high"])
        past = rng.randint(case["past_low"], case["past_high"])
        out.append((q, n, kv, past + n))
        q += n
        kv += past + n + (rng.randint(0, 7) if case["past_high"] else 0)
    return np.asarray(out, dtype=np.uint32)


def scale(case):
    """The encoders' heads are RMS-normed and score unscaled; the other layouts divide by sqrt(head dim)."""
    return 1.0 if case["head_dim"] >= 256 else case["head_dim"] ** -0.5


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def attention_inputs(case, seed):
    g, t, seqs = generator(seed), TYPES[case["type"]], sequences(case)
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["head_dim"]
    rows, kv_rows = int(seqs[-1, 0] + seqs[-1, 1]), int(seqs[-1, 2] + seqs[-1, 3])

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(t)

    if case.get("fused"):
        qkv = normal(rows, heads + 2 * kv_heads, hd)
        q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
    else:
        q, k, v = normal(rows, heads, hd), normal(kv_rows, kv_heads, hd), normal(kv_rows, kv_heads, hd)
    s = dict(kind=case["kind"], case=dict(case), q=q, k=k, v=v, seqs=seqs)
    if case["kind"] == "prefix":
        s["prefix_k"], s["prefix_v"] = (normal(case["prefix"], kv_heads, hd) for _ in range(2))
    return s


def q4_rows(rng, kind, rows, width):
    """GGUF rows: blocks of an fp16 scale (and, Q4_1, an fp16 minimum) and 32 quants uniform in 0 .. 15, the
    low nibbles of the 16 bytes first."""
    blocks = np.zeros((rows * width // 32, BLOCK_BYTES[kind]), np.uint8)
    d = (np.abs(rng.normal(0.0, 0.02, len(blocks))) / 8).astype(np.float16)
    blocks[:, :2] = d.view(np.uint8).reshape(-1, 2)
    if kind == "q4_1":
        m = (d.astype(np.float32) * rng.uniform(-9.0, -6.0, len(blocks))).astype(np.float16)
        blocks[:, 2:4] = m.view(np.uint8).reshape(-1, 2)
    blocks[:, -16:] = rng.integers(0, 256, (len(blocks), 16), dtype=np.uint8)
    return blocks


def q4_inputs(case, seed):
    rng, g = np.random.default_rng(seed), generator(seed)
    w = [q4_rows(rng, case["weights"], case["features"], case["width"]) for _ in range(2 if case["geglu"] else 1)]
    x = torch.randn(case["rows"], case["width"], generator=g, device="cuda").to(TYPES[case["x"]])
    return w, x


HELD = {}


def library():
    if "library" not in HELD:
        sys.path.insert(0, os.path.abspath("gemma-embed-swift_amd"))
        import gemma_embed
        HELD["library"], HELD["context"] = gemma_embed, gemma_embed.Context.create(0)
    return HELD["library"], HELD["context"]


class Matrix:
    """A 4-bit weight matrix in device memory, given back with its state."""

    def __init__(self, context, blocks, kind, rows, cols):
        self.context, self.handle = context, context.q4_create(blocks, GGUF_TYPES[kind], rows, cols)

    def __del__(self):
        self.context.q4_destroy(self.handle)


def prepare(case, seed):
    if case["kind"] == "q4":
        w, x = q4_inputs(case, seed)
        s = dict(kind="q4", case=dict(case), x=x)
        if own:
            _, c = library()
            s["w"] = [Matrix(c, b, case["weights"], case["features"], case["width"]) for b in w]
            s["out"] = torch.empty(case["rows"], case["features"], device="cuda", dtype=TYPES[case["y"]])
        else:
            # the file's planes, still in 4 bits
            s["w"] = [dict(quants=torch.from_numpy(b[:, -16:].copy()).cuda(),
                           scales=torch.from_numpy(b[:, :-16].copy().view(np.float16)).cuda()) for b in w]
        return s
    s = attention_inputs(case, seed)
    if own:
        ge, _ = library()
        s["out"] = torch.empty(s["q"].shape, device="cuda", dtype=s["q"].dtype)
        s["shape"] = ge.attention_shape(GGUF_TYPES[case["type"]], case["heads"], case["kv_heads"], case["head_dim"],
                                        q_rows=s["q"].shape[0], kv_rows=s["k"].shape[0], scale=scale(case),
                                        window=case["window"], q_stride=s["q"].stride(0), k_stride=s["k"].stride(0),
                                        v_stride=s["v"].stride(0), out_stride=s["out"].stride(0))
    return s


# ---------------------------------------------------------------------------- one pass


def run(s):
    if not own:
        return {"causal": plain_causal, "prefix": plain_prefix, "q4": plain_q4}[s["kind"]](s)
    _, c = library()
    if s["kind"] == "causal":
        c.attention_causal(s["shape"], s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["seqs"],
                           s["out"].data_ptr())
    elif s["kind"] == "prefix":
        c.attention_prefix(s["shape"], s["q"].data_ptr(), s["prefix_k"].data_ptr(), s["prefix_v"].data_ptr(),
                           s["case"]["prefix"], s["k"].data_ptr(), s["v"].data_ptr(), s["seqs"], s["out"].data_ptr())
    else:
        k = s["case"]
        call = (s["x"].data_ptr(), GGUF_TYPES[k["x"]], k["rows"], s["out"].data_ptr(), GGUF_TYPES[k["y"]])
        if k["geglu"]:
            c.gemv_q4_geglu(s["w"][0].handle, s["w"][1].handle, *call)
        else:
            c.gemv_q4(s["w"][0].handle, *call)
    return s["out"]


def heads_first(x, group):
    """[rows][heads][hd] as fp32 [KV heads][rows * group][hd]."""
    rows, heads, hd = x.shape
    return x.float().reshape(rows, heads // group, group, hd).permute(1, 0, 2, 3).reshape(heads // group, rows * group, hd)


def plain_scores(q, k, case, position, first):
    """Scaled scores of query rows at `position` (one per row) against keys at positions first, first + 1, ...;
    -inf where a key is not visible."""
    s = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(scale(case))
    j = first + torch.arange(k.shape[1], device=k.device)
    hidden = j[None, :] > position[:, None]
    if case["window"]:
        hidden |= j[None, :] <= position[:, None] - case["window"]
    return s.masked_fill_(hidden, -math.inf)


def plain_causal(s):
    case, out = s["case"], torch.zeros(s["q"].shape, device="cuda", dtype=s["q"].dtype)
    g, kv_heads = case["heads"] // case["kv_heads"], case["kv_heads"]
    for q0, n, k0, m in s["seqs"].tolist():
        q, k, v = heads_first(s["q"][q0:q0 + n], g), heads_first(s["k"][k0:k0 + m], 1), heads_first(s["v"][k0:k0 + m], 1)
        position = (torch.arange(n, device="cuda") + (m - n)).repeat_interleave(g)
        o = torch.empty_like(q)
        step = max(1, (1 << 30) // (n * g * m))  # KV heads at once: scores of 4 GiB at most
        for h in range(0, kv_heads, step):
            p = plain_scores(q[h:h + step], k[h:h + step], case, position, 0)
            top = p.amax(-1, keepdim=True).clamp_(min=-3e38)
            p = p.sub_(top).exp_()
            total = p.sum(-1, keepdim=True)
            o[h:h + step] = torch.matmul(p, v[h:h + step]).div_(total.clamp_(min=1e-38))
        out[q0:q0 + n] = o.reshape(kv_heads, n, g, -1).permute(1, 0, 2, 3).reshape(n, case["heads"], -1).to(out.dtype)
    return out


def plain_prefix(s):
    case, out = s["case"], torch.zeros(s["q"].shape, device="cuda", dtype=s["q"].dtype)
    g, kv_heads, first = case["heads"] // case["kv_heads"], case["kv_heads"], case["prefix"]
    q, seqs = heads_first(s["q"], g), s["seqs"].tolist()
    pk, pv = heads_first(s["prefix_k"], 1), heads_first(s["prefix_v"], 1)
    position = torch.cat([torch.arange(n, device="cuda") + (first + m - n) for _, n, _, m in seqs]).repeat_interleave(g)
    # the prefix's part for every row at once: maximum, sum and unnormalised result
    shared = plain_scores(q, pk, case, position, 0)
    top = shared.amax(-1, keepdim=True)
    shared = shared.sub_(top.clamp(min=-3e38)).exp_()
    total, o = shared.sum(-1, keepdim=True), torch.matmul(shared, pv)
    for q0, n, k0, m in seqs:
        rows = slice(q0 * g, (q0 + n) * g)
        k, v = heads_first(s["k"][k0:k0 + m], 1), heads_first(s["v"][k0:k0 + m], 1)
        p = plain_scores(q[:, rows], k, case, position[rows], first)
        both = torch.maximum(top[:, rows], p.amax(-1, keepdim=True)).clamp_(min=-3e38)
        fade = (top[:, rows].clamp(min=-3e38) - both).exp_()
        p = p.sub_(both).exp_()
        y = torch.matmul(p, v).add_(o[:, rows] * fade)
        y = y.div_((p.sum(-1, keepdim=True) + total[:, rows] * fade).clamp_(min=1e-38))
        out[q0:q0 + n] = y.reshape(kv_heads, n, g, -1).permute(1, 0, 2, 3).reshape(n, case["heads"], -1).to(out.dtype)
    return out


def gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


def plain_q4(s):
    case, y = s["case"], []
    for w in s["w"]:
        q = torch.cat([w["quants"] & 15, w["quants"] >> 4], 1).float()
        d = w["scales"].float()
        m = d[:, 1:] if case["weights"] == "q4_1" else -8.0 * d
        y.append(s["x"].float() @ (q * d[:, :1] + m).reshape(case["features"], case["width"]).T)
    return (gelu(y[0]) * y[1] if case["geglu"] else y[0]).to(TYPES[case["y"]])


# ---------------------------------------------------------------------------- necessary work


def pairs(n, position, first, keys, window):
    """Visible (query, key) pairs of n queries at positions position, position + 1, ... and `keys` keys from
    position `first` on."""
    p = position + np.arange(n, dtype=np.int64)
    low = np.maximum(first, p - window + 1) if window else np.full(n, first, np.int64)
    return int(np.maximum(np.minimum(p, first + keys - 1) - low + 1, 0).sum())


def work(case):
    if case["kind"] == "q4":
        rows, k, f, n = case["rows"], case["width"], case["features"], 2 if case["geglu"] else 1
        return dict(bytes=n * f * k * BLOCK_BYTES[case["weights"]] / 32 + rows * (2 * k + f * (4 if case["y"] == "f32" else 2)),
                    flops=2 * n * rows * k * f)
    seqs, hd, window = sequences(case).tolist(), case["head_dim"], case["window"]
    first = case.get("prefix", 0)
    rows, seen, keys = sum(n for _, n, _, _ in seqs), 0, 0
    for _, n, _, m in seqs:
        seen += pairs(n, first + m - n, 0, first, window) + pairs(n, first + m - n, first, m, window)
        keys += min(m, n + window - 1) if window else m
    # of the prefix, the rows some query sees: with a window, those within it of the earliest query
    if first:
        keys += min(first, max(0, window - 1 - min(m - n for _, n, _, m in seqs))) if window else first
    return dict(bytes=2 * hd * (2 * case["heads"] * rows + 2 * case["kv_heads"] * keys), flops=4 * hd * case["heads"] * seen)


# ---------------------------------------------------------------------------- the same in 64 bits


def exact(case, seed):
    if case["kind"] == "q4":
        blocks, x = q4_inputs(case, seed)
        y = []
        for b in blocks:
            d = torch.from_numpy(b[:, :2].copy().view(np.float16).astype(np.float64)).cuda()
            codes = torch.from_numpy(b[:, -16:].astype(np.int64)).cuda()
            w = torch.empty(len(b), 32, dtype=torch.float64, device="cuda")
            if case["weights"] == "q4_0":
                w[:, :16], w[:, 16:] = (codes % 16 - 8) * d, (codes // 16 - 8) * d
            else:
                least = torch.from_numpy(b[:, 2:4].copy().view(np.float16).astype(np.float64)).cuda()
                w[:, :16], w[:, 16:] = codes % 16 * d + least, codes // 16 * d + least
            y.append(x.double() @ w.reshape(case["features"], case["width"]).T)
        return gelu(y[0]) * y[1] if case["geglu"] else y[0]
    s = attention_inputs(case, seed)
    out, group = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), case["heads"] // case["kv_heads"]
    for q0, n, k0, m in s["seqs"].tolist():
        for h in range(case["heads"]):
            k, v = s["k"][k0:k0 + m, h // group].double(), s["v"][k0:k0 + m, h // group].double()
            if case["kind"] == "prefix":
                k = torch.cat([s["prefix_k"][:, h // group].double(), k])
                v = torch.cat([s["prefix_v"][:, h // group].double(), v])
            logits = (s["q"][q0:q0 + n, h].double() @ k.T) * scale(case)
            ahead = torch.arange(len(k), device="cuda")[None, :] - torch.arange(n, device="cuda")[:, None] - (len(k) - n)
            logits.masked_fill_(ahead > 0, -math.inf)
            if case["window"]:
                logits.masked_fill_(ahead <= -case["window"], -math.inf)
            out[q0:q0 + n, h] = torch.softmax(logits, -1).nan_to_num_(nan=0.0) @ v
    return out
