"""The operators of a paged cache of keys and values, each as one call: norms and rotary positions of query and
key heads, appending a call's tokens to the pages, and attention of chunks and single tokens over the pages.

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
GGUF_TYPES = {"f32": 0, "f16": 1, "bf16": 30}
LAYOUTS = {"halves": 0, "pairs": 1}
SCALINGS = {"plain": 0, "linear": 1, "by_turns": 2}
# Query heads, KV heads, head dim: the two text encoders' layers (window 512 and 1024 on the sliding
# ones), then the usual grouped, ungrouped and narrow layouts.
HEADS = [(3, 1, 256), (4, 2, 256), (4, 1, 512), (2, 1, 128), (32, 8, 128), (6, 6, 128), (16, 8, 64), (12, 4, 64)]
# Layouts of heads that are rotated and cached, but not attended to here.
ODD_HEADS = [(5, 1, 80), (6, 2, 96), (4, 4, 40), (7, 1, 72), (2, 2, 34)]
PAGES = [8, 16, 32, 64, 128, 256]
# A rotation: rotated elements of a head (0: all), layout, base, scaling, factor, trained positions, magnitude.
PLAIN = dict(dims=0, layout="halves", base=1e4, scaling="plain", factor=1.0, trained=0, magnitude=1.0)
LONG = dict(dims=0, layout="halves", base=5e5, scaling="by_turns", factor=8.0, trained=8192, magnitude=1.0)
STRETCHED = dict(dims=0, layout="pairs", base=1e4, scaling="linear", factor=4.0, trained=0, magnitude=1.0)
LOW_TURNS, HIGH_TURNS = 1.0, 4.0
EPS = 1e-6


def listed():
    return [
        # One text's next token: its projection in fp32, normed and rotated as the encoder's heads are. All latency.
        dict(name="rotate_token", kind="rotate", input="f32", type="f16", rows=1, heads=3, kv_heads=1, head_dim=256,
             normed=True, position_low=2000, position_high=2000, fused=True, **dict(PLAIN, base=1e6)),
        # A few texts' tokens with neighbouring elements paired and half of each head rotated.
        dict(name="rotate_pairs", kind="rotate", input="f16", type="f16", rows=777, heads=12, kv_heads=4, head_dim=64,
             normed=True, position_low=0, position_high=2047, fused=True, **dict(STRETCHED, dims=32)),
        # A long prompt of grouped heads, positions far past those the model was trained on.
        dict(name="rotate_prompt", kind="rotate", input="bf16", type="bf16", rows=16384, heads=32, kv_heads=8,
             head_dim=128, normed=False, position_low=100000, position_high=116383, fused=True, **LONG),
        # One token of the reference architecture's global layers into the cache.
        dict(name="append_token", kind="append", input="f32", type="f16", sequences=1, low=1, high=1, past_low=300,
             past_high=300, heads=4, kv_heads=1, head_dim=512, normed=True, page=64, fused=False, **dict(PLAIN, base=1e6)),
        # A serving step: one token of each of 128 texts.
        dict(name="append_steps", kind="append", input="bf16", type="bf16", sequences=128, low=1, high=1, past_low=100,
             past_high=900, heads=32, kv_heads=8, head_dim=128, normed=False, page=16, fused=True, **LONG),
        # A ragged pack of passages on a sliding-window layer, from the projection's fp32 rows.
        dict(name="append_passages", kind="append", input="f32", type="bf16", sequences=9, low=130, high=997, past_low=0,
             past_high=0, heads=3, kv_heads=1, head_dim=256, normed=True, page=16, fused=True, **PLAIN),
        # A chapter read behind another one.
        dict(name="append_chapter", kind="append", input="f16", type="f16", sequences=1, low=8192, high=8192,
             past_low=8000, past_high=8000, heads=32, kv_heads=8, head_dim=128, normed=True, page=128, fused=True, **LONG),
        # One text's next token on a sliding-window layer: all latency.
        dict(name="paged_token", kind="attention", type="f16", sequences=1, low=1, high=1, past_low=700, past_high=700,
             heads=3, kv_heads=1, head_dim=256, window=512, cap=0.0, page=16),
        # A serving step: one token for each of 64 texts over caches of different lengths.
        dict(name="paged_steps", kind="attention", type="bf16", sequences=64, low=1, high=1, past_low=100, past_high=8000,
             heads=32, kv_heads=8, head_dim=128, window=0, cap=0.0, page=16),
        # Documents read in chunks.
        dict(name="paged_chunks", kind="attention", type="f16", sequences=5, low=301, high=700, past_low=2000,
             past_high=9000, heads=16, kv_heads=8, head_dim=64, window=0, cap=0.0, page=64),
        # Chunks on a sliding-window layer whose scores are capped.
        dict(name="paged_capped", kind="attention", type="bf16", sequences=3, low=500, high=1500, past_low=1000,
             past_high=4000, heads=4, kv_heads=2, head_dim=256, window=1024, cap=50.0, page=32),
        # A chapter read behind another one.
        dict(name="paged_chapter", kind="attention", type="bf16", sequences=1, low=8192, high=8192, past_low=8000,
             past_high=8000, heads=32, kv_heads=8, head_dim=128, window=0, cap=0.0, page=128),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["rotate", "append", "attention", "attention"])
    case = dict(kind=kind, type=rng.choice(["f16", "bf16"]))
    if kind != "rotate":
        case["page"] = rng.choice(PAGES)
        form = rng.choice(["prompt", "chunk", "token"])
        high = 1 if form == "token" else spread(2, 4096 if form == "prompt" else 512)
        past = 0 if form == "prompt" else spread(16, 32768 if kind == "attention" else 4096)
        case.update(sequences=min(spread(1, 128), max(1, 8192 // high), max(1, 131072 // (past + high))),
                    low=max(1, high // 2), high=high, past_low=past // 8, past_high=past)
    if kind == "attention":
        case.update(window=rng.choice([0, 0, 512, 1024, spread(1, 4096)]), cap=rng.choice([0.0, 0.0, 30.0, 50.0]))
        case["heads"], case["kv_heads"], case["head_dim"] = rng.choice(HEADS)
        return case
    heads, kv_heads, head_dim = rng.choice(HEADS + ODD_HEADS)
    if kind == "rotate":
        first = rng.choice([0, spread(1, 1 << 20)])
        case.update(rows=min(spread(1, 16384), (1 << 26) // (heads * head_dim)), position_low=first, position_high=first + spread(1, 100000))
    case.update(rng.choice([PLAIN, LONG, STRETCHED]))
    case.update(input=rng.choice(["f32", case["type"]]), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                normed=rng.random() < 0.5, fused=head_dim < 512 and rng.random() < 0.5,
                dims=rng.choice([0, 0, head_dim // 2, 2 * rng.randint(1, head_dim // 2)]),
                layout=rng.choice(["halves", "pairs"]), base=rng.choice([1e4, 5e5, 1e6]))
    if case["scaling"] != "plain":
        case.update(factor=rng.choice([2.0, 8.0, 32.0]), magnitude=rng.choice([1.0, 1.2]))
    return case


# ---------------------------------------------------------------------------- inputs


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def fixed(case):
    """A generator that the case alone decides: lengths and pages are the same for every seed."""
    return random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))


def sequences(case):
    """(q_start, q_len, slot, kv_len) of each text: its new rows, packed back to back, its row of the page table
    and its keys, the new ones among them."""
    rng, out, at = fixed(case), [], 0
    for slot in range(case["sequences"]):
        n = rng.randint(case["low"], case["high"])
        out.append((at, n, slot, n + rng.randint(case["past_low"], case["past_high"])))
        at += n
    return np.asarray(out, dtype=np.uint32)


def pages(case):
    """(table [slots][pages of the longest] int32, -1 past a text's own; pages in the pool): the pages of a pool
    that has been in use for a while, in no order."""
    seqs, p = sequences(case), case["page"]
    counts = [-(-int(m) // p) for m in seqs[:, 3]]
    spare = sum(counts) // 16 + 3
    order = list(range(sum(counts) + spare))
    fixed(case).shuffle(order)
    table = np.full((len(counts), max(counts)), -1, np.int32)
    at = 0
    for slot, n in enumerate(counts):
        table[slot, :n] = order[at:at + n]
        at += n
    return table, len(order)


def scale(case):
    """The encoders' heads are RMS-normed and score unscaled; the other layouts divide by sqrt(head dim)."""
    return 1.0 if case["head_dim"] >= 256 else case["head_dim"] ** -0.5


def inputs(case, seed):
    """The tensors of one call, by name."""
    g, t = generator(seed), TYPES[case["type"]]
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["head_dim"]

    def normal(*shape, to=t):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(to)

    s = {}
    if case["kind"] == "attention":
        s["q"] = normal(int(sequences(case)[:, 1].sum()), heads, hd)
    else:
        rows = case["rows"] if case["kind"] == "rotate" else int(sequences(case)[:, 1].sum())
        kinds = [heads, kv_heads, kv_heads]
        if case["fused"]:
            s["q"], s["k"], s["v"] = normal(rows, sum(kinds), hd, to=TYPES[case["input"]]).split(kinds, 1)
        else:
            s["q"], s["k"], s["v"] = (normal(rows, h, hd, to=TYPES[case["input"]]) for h in kinds)
        if case["normed"]:
            s["q_norm"], s["k_norm"] = (1 + 0.1 * normal(hd, to=torch.float32) for _ in range(2))
    if case["kind"] == "rotate":
        s["positions"] = torch.randint(case["position_low"], case["position_high"] + 1, (case["rows"],), generator=g,
                                       device="cuda", dtype=torch.int32)
    else:
        _, n = pages(case)
        s["k_pages"], s["v_pages"] = (normal(n, kv_heads, case["page"], hd) for _ in range(2))
    return s


HELD = {}


def library():
    if "library" not in HELD:
        sys.path.insert(0, os.path.abspath("gemma-embed-swift_amd"))
        import gemma_embed
        HELD["library"], HELD["context"] = gemma_embed, gemma_embed.Context.create(0)
    return HELD["library"], HELD["context"]


class Handle:
    """A handle of the library's, given back with its state."""

    def __init__(self, value, destroy):
        self.value, self.destroy = value, destroy

    def __del__(self):
        self.destroy(self.value)


def prepare(case, seed):
    s = dict(inputs(case, seed), kind=case["kind"], case=dict(case))
    hd = case["head_dim"]
    if case["kind"] != "rotate":
        table, n = pages(case)
        s["seqs"] = sequences(case)
        if not own:
            s["table"] = torch.from_numpy(table.astype(np.int64)).cuda()
    if not own:
        return s
    ge, c = library()
    if case["kind"] != "rotate":
        h = c.page_table_create(table.shape[0], table.shape[1], case["page"], n)
        s["table"] = Handle(h, c.page_table_destroy)
        slots, at = np.nonzero(table >= 0)
        c.page_table_set(h, np.stack([slots, at, table[slots, at]], 1))
    s["q_out"] = torch.empty(s["q"].shape, device="cuda", dtype=TYPES[case["type"]])
    if case["kind"] == "attention":
        s["shape"] = ge.paged_shape(GGUF_TYPES[case["type"]], case["heads"], case["kv_heads"], hd,
                                    q_rows=s["q"].shape[0], scale=scale(case), window=case["window"], cap=case["cap"],
                                    q_stride=s["q"].stride(0))
        return s
    s["rotary"] = Handle(c.rotary_create(case["dims"] or hd, case["base"], layout=LAYOUTS[case["layout"]],
                                         scaling=SCALINGS[case["scaling"]], factor=case["factor"], low_turns=LOW_TURNS,
                                         high_turns=HIGH_TURNS, trained=case["trained"], magnitude=case["magnitude"]),
                         c.rotary_destroy)
    normed = (ge.GE_NORM_Q | ge.GE_NORM_K) if case["normed"] else 0
    if case["kind"] == "rotate":
        s["k_out"] = torch.empty(s["k"].shape, device="cuda", dtype=TYPES[case["type"]])
    elif case["normed"]:
        normed |= ge.GE_NORM_V
    s["shape"] = ge.heads_shape(GGUF_TYPES[case["input"]], GGUF_TYPES[case["type"]], case["heads"], case["kv_heads"], hd,
                                rows=s["q"].shape[0], normed=normed, eps=EPS, q_stride=s["q"].stride(0),
                                k_stride=s["k"].stride(0), v_stride=s["v"].stride(0))
    return s


# ---------------------------------------------------------------------------- one pass


def run(s):
    if not own:
        return {"rotate": plain_rotate, "append": plain_append, "attention": plain_attention}[s["kind"]](s)
    _, c = library()
    if s["kind"] == "attention":
        c.attention_paged(s["shape"], s["q"].data_ptr(), s["table"].value, s["k_pages"].data_ptr(), s["v_pages"].data_ptr(),
                          s["seqs"], s["q_out"].data_ptr())
        return s["q_out"]
    q_norm, k_norm = (s["q_norm"].data_ptr(), s["k_norm"].data_ptr()) if s["case"]["normed"] else (None, None)
    if s["kind"] == "rotate":
        c.rotate_heads(s["shape"], s["rotary"].value, s["q"].data_ptr(), s["k"].data_ptr(), q_norm, k_norm,
                       s["positions"].data_ptr(), s["q_out"].data_ptr(), s["k_out"].data_ptr())
        return [s["q_out"], s["k_out"]]
    c.paged_append(s["shape"], s["rotary"].value, s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), q_norm, k_norm,
                   None, s["table"].value, s["seqs"], s["q_out"].data_ptr(), s["k_pages"].data_ptr(), s["v_pages"].data_ptr())
    return [s["q_out"], s["k_pages"], s["v_pages"]]


def plain_norm(x, w):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return y if w is None else y * w


def plain_turned(x, case, angles):
    """x [rows][heads][hd] with its first elements rotated by angles [rows][pairs] (64 bits)."""
    dims = case["dims"] or case["head_dim"]
    cos = (torch.cos(angles).float() * case["magnitude"])[:, None]
    sin = (torch.sin(angles).float() * case["magnitude"])[:, None]
    halves = case["layout"] == "halves"
    a, b = (x[..., :dims // 2], x[..., dims // 2:dims]) if halves else (x[..., 0:dims:2], x[..., 1:dims:2])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([a, b], -1) if halves else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., dims:]], -1)


def plain_angles(case, positions):
    dims = case["dims"] or case["head_dim"]
    f = torch.exp(torch.arange(dims // 2, device="cuda", dtype=torch.float64) * (-2.0 / dims * math.log(case["base"])))
    if case["scaling"] == "linear":
        f = f / case["factor"]
    elif case["scaling"] == "by_turns":
        turns = f * (case["trained"] / (2 * math.pi))
        w = ((turns - LOW_TURNS) / (HIGH_TURNS - LOW_TURNS)).clamp(0.0, 1.0)
        f = f * (w + (1.0 - w) / case["factor"])
    return positions.double()[:, None] * f


def plain_rotate(s):
    case, out = s["case"], []
    angles = plain_angles(case, s["positions"])
    for x, w in (("q", "q_norm"), ("k", "k_norm")):
        y = s[x].float()
        if case["normed"]:
            y = plain_norm(y, s[w])
        out.append(plain_turned(y, case, angles).to(TYPES[case["type"]]))
    return out


def plain_append(s):
    case, seqs = s["case"], s["seqs"].astype(np.int64)
    at = np.concatenate([np.arange(m - n, m) for _, n, _, m in seqs])
    at, slot = torch.from_numpy(at).cuda(), torch.from_numpy(np.repeat(seqs[:, 2], seqs[:, 1])).cuda()
    page, row = s["table"][slot, at // case["page"]], at % case["page"]
    angles = plain_angles(case, at)
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if case["normed"]:
        q, k, v = plain_norm(q, s["q_norm"]), plain_norm(k, s["k_norm"]), plain_norm(v, None)
    t = TYPES[case["type"]]
    s["k_pages"][page, :, row] = plain_turned(k, case, angles).to(t)
    s["v_pages"][page, :, row] = v.to(t)
    return [plain_turned(q, case, angles).to(t), s["k_pages"], s["v_pages"]]


def plain_attention(s):
    case, out = s["case"], torch.zeros(s["q"].shape, device="cuda", dtype=s["q"].dtype)
    kv_heads, hd, g = case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]

    def keys(pool, ids, first, end):  # [pages][KV heads][rows][hd] as fp32 [KV heads][keys][hd]
        return pool[ids].permute(1, 0, 2, 3).reshape(kv_heads, -1, hd)[:, first:end].float()

    for q0, n, slot, m in s["seqs"].tolist():
        low = max(0, m - n - case["window"] + 1) if case["window"] else 0  # the first key that a row sees
        first = low // case["page"]
        ids = s["table"][slot, first:-(-m // case["page"])]
        low, end = low - first * case["page"], m - first * case["page"]
        k, v = keys(s["k_pages"], ids, low, end), keys(s["v_pages"], ids, low, end)
        q = s["q"][q0:q0 + n].float().reshape(n, kv_heads, g, hd).permute(1, 0, 2, 3).reshape(kv_heads, n * g, hd)
        position = (torch.arange(n, device="cuda") + (m - n)).repeat_interleave(g)
        j = m - k.shape[1] + torch.arange(k.shape[1], device="cuda")
        hidden = j[None, :] > position[:, None]
        if case["window"]:
            hidden |= j[None, :] <= position[:, None] - case["window"]
        o = torch.empty_like(q)
        step = max(1, (1 << 30) // (n * g * k.shape[1]))  # KV heads at once: scores of 4 GiB at most
        for h in range(0, kv_heads, step):
            p = torch.matmul(q[h:h + step], k[h:h + step].transpose(1, 2).contiguous()).mul_(scale(case))
            if case["cap"]:
                p = p.div_(case["cap"]).tanh_().mul_(case["cap"])
            p = p.masked_fill_(hidden, -math.inf)
            p = p.sub_(p.amax(-1, keepdim=True)).exp_()
            total = p.sum(-1, keepdim=True)
            o[h:h + step] = torch.matmul(p, v[h:h + step]).div_(total)
        out[q0:q0 + n] = o.reshape(kv_heads, n, g, hd).permute(1, 0, 2, 3).reshape(n, case["heads"], hd).to(out.dtype)
    return out


# ---------------------------------------------------------------------------- necessary work


def work(case):
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "attention":
        window, rows, seen, keys, ids = case["window"], 0, 0, 0, 0
        for _, n, _, m in sequences(case).tolist():
            last = m - n + np.arange(n, dtype=np.int64)
            low = np.maximum(0, last - window + 1) if window else np.zeros(n, np.int64)
            seen += int((last - low + 1).sum())
            keys += m - int(low[0])
            ids += -(-m // case["page"]) - int(low[0]) // case["page"]
            rows += n
        return dict(bytes=2 * hd * (2 * heads * rows + 2 * kv_heads * keys) + 4 * ids, flops=4 * hd * heads * seen)
    rotate = case["kind"] == "rotate"
    rows = case["rows"] if rotate else int(sequences(case)[:, 1].sum())
    turned = rows * (heads + kv_heads)
    rows_of = turned if rotate else rows * (heads + 2 * kv_heads)
    size = 4 if case["input"] == "f32" else 2
    return dict(bytes=rows_of * hd * (size + 2) + 4 * rows,
                flops=turned * 3 * (case["dims"] or hd) + (rows_of * 4 * hd if case["normed"] else 0))


# ---------------------------------------------------------------------------- the same in 64 bits


def exact_rows(case, x, w, positions):
    """Rows [n][heads][hd] normed by w (None: not; True: with no weight) and rotated (positions None: not)."""
    y = x.double()
    if w is not None:
        y = y / (y.square().sum(-1, keepdim=True) / case["head_dim"] + EPS).sqrt()
        y = y if w is True else y * w.double()
    if positions is None:
        return y
    dims, out = case["dims"] or case["head_dim"], y.clone()
    for i in range(dims // 2):
        f = float(case["base"]) ** (-2.0 * i / dims)
        if case["scaling"] == "linear":
            f /= case["factor"]
        if case["scaling"] == "by_turns":
            part = min(1.0, max(0.0, (case["trained"] * f / (2.0 * math.pi) - LOW_TURNS) / (HIGH_TURNS - LOW_TURNS)))
            f = part * f + (1.0 - part) * f / case["factor"]
        a, b = (i, dims // 2 + i) if case["layout"] == "halves" else (2 * i, 2 * i + 1)
        c = torch.polar(torch.full_like(positions, case["magnitude"], dtype=torch.float64), positions.double() * f)[:, None]
        z = torch.complex(y[..., a], y[..., b]) * c
        out[..., a], out[..., b] = z.real, z.imag
    return out


def exact(case, seed):
    s = inputs(case, seed)
    if case["kind"] == "rotate":
        return [exact_rows(case, s[x], s.get(x + "_norm"), s["positions"]) for x in ("q", "k")]
    (table, _), out = pages(case), None
    p, group = case["page"], case["heads"] // case["kv_heads"]
    if case["kind"] == "append":
        q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        pools = [s["k_pages"].double(), s["v_pages"].double()]
        for q0, n, slot, m in sequences(case).tolist():
            rows, at = slice(q0, q0 + n), torch.arange(m - n, m, device="cuda")
            q[rows] = exact_rows(case, s["q"][rows], s.get("q_norm"), at)
            new = [exact_rows(case, s["k"][rows], s.get("k_norm"), at),
                   exact_rows(case, s["v"][rows], True if case["normed"] else None, None)]
            for j0 in range((m - n) // p * p, m, p):  # page by page
                lo, hi = max(j0, m - n), min(j0 + p, m)
                for pool, x in zip(pools, new):
                    pool[int(table[slot, j0 // p]), :, lo - j0:hi - j0] = x[lo - (m - n):hi - (m - n)].transpose(0, 1)
        return [q] + pools
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for q0, n, slot, m in sequences(case).tolist():
        low = max(0, m - n - case["window"] + 1) if case["window"] else 0
        j = torch.arange(low, m, device="cuda")
        page, row = torch.from_numpy(table[slot].astype(np.int64)).cuda()[j // p], j % p
        ahead = j[None, :] - (m - n) - torch.arange(n, device="cuda")[:, None]
        hidden = ahead > 0
        if case["window"]:
            hidden |= ahead <= -case["window"]
        for h in range(case["heads"]):
            k, v = s["k_pages"][page, h // group, row].double(), s["v_pages"][page, h // group, row].double()
            logits = (s["q"][q0:q0 + n, h].double() @ k.T) * scale(case)
            if case["cap"]:
                logits = torch.tanh(logits / case["cap"]) * case["cap"]
            out[q0:q0 + n, h] = torch.softmax(logits.masked_fill(hidden, -math.inf), -1) @ v
    return out
