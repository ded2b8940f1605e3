"""The attention of causal models on the host HIP runtime (host_hip.cpp): what a call's plan gives its
kernels, and what a call refuses. Run by tests/test_causal_plan.py in a process of its own, whose GE_LIBRARY
is the library's objects over that runtime."""
import ctypes as C
import random

import numpy as np
import pytest

import gemma_embed as ge

P, I = C.c_void_p, C.c_int
LAUNCH = C.CFUNCTYPE(None, C.c_char_p, C.POINTER(P))
lib = ge.lib
lib.host_hip_pending.restype = C.c_uint64
lib.host_hip_fail.argtypes = [C.c_char_p, I]
lib.host_hip_on_launch.argtypes = [LAUNCH]
DIRECT = 0xffffffff


class Item(C.Structure):
    """CausalItem, causal.hpp"""
    _fields_ = [(n, C.c_uint32) for n in ("q_token", "row0", "n_rows", "key0", "k_lo", "k_hi")] + \
        [("shift", C.c_int32)] + [(n, C.c_uint32) for n in ("part", "narrow")]


class Join(C.Structure):
    """CausalJoin"""
    _fields_ = [(n, C.c_uint32) for n in ("q_token", "row0", "n_rows")] + \
        [(n, C.c_uint32 * 2) for n in ("part", "stride", "splits")]


class Args(C.Structure):
    """CausalArgs"""
    _fields_ = [(n, P) for n in ("q", "k", "v", "prefix_k", "prefix_v", "out")] + \
        [("items", C.POINTER(Item)), ("joins", C.POINTER(Join)), ("part_o", P), ("part_ml", P)] + \
        [(n, C.c_int64) for n in ("q_stride", "k_stride", "v_stride", "out_stride")] + [("part_rows", C.c_size_t)] + \
        [(n, I) for n in ("n_items", "n_joins", "join_rows", "group", "kv_heads", "window", "prefix_len")] + [("c", C.c_float), ("q_flip", C.c_uint32)]


class Inline(C.Structure):
    """CausalInline: the lists of a call that has few of both"""
    _fields_ = [("items", Item * 48), ("joins", Join * 40)]


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def memory(ctx):
    return ctx.alloc(1 << 16)


class Call:
    """The items and joins of one call, copied as its launches are made."""

    def __init__(self):
        self.items, self.joins, self.args, self.error, self.names = [], [], None, None, []

    def __enter__(self):
        def on_launch(name, args):
            try:
                name, a = name.decode(), C.cast(args[0], C.POINTER(Args))[0]
                few = C.cast(args[1], C.POINTER(Inline))[0]
                self.names.append(name)
                self.args = {f: getattr(a, f) for f, _ in Args._fields_ if f not in ("items", "joins")}
                if "causal_join_kernel" in name:
                    assert bool(a.joins) == (a.n_joins > 40 or a.n_items > 48)
                    self.joins = [Join.from_buffer_copy((a.joins or few.joins)[i]) for i in range(a.n_joins)]
                else:
                    assert bool(a.items) == (a.n_joins > 40 or a.n_items > 48)
                    self.items = [Item.from_buffer_copy((a.items or few.items)[i]) for i in range(a.n_items)]
            except BaseException as e:  # noqa: BLE001
                self.error = self.error or e
        self.callback = LAUNCH(on_launch)
        lib.host_hip_on_launch(self.callback)
        return self

    def __exit__(self, *exc):
        lib.host_hip_on_launch(LAUNCH())
        if self.error and not exc[0]:
            raise self.error


def call(ctx, memory, seqs, heads, kv_heads, hd, window=0, prefix=0, **kw):
    q_rows = max([s[0] + s[1] for s in seqs] + [0])
    kv_rows = max([s[2] + s[3] for s in seqs] + [0])
    shape = ge.attention_shape(kw.pop("type", ge.GE_TYPE_F16), heads, kv_heads, hd, kw.pop("q_rows", q_rows),
                               kw.pop("kv_rows", kv_rows), window=window, **kw)
    with Call() as got:
        if prefix:
            ctx.attention_prefix(shape, memory, memory, memory, prefix, memory, memory, seqs, memory)
        else:
            ctx.attention_causal(shape, memory, memory, memory, seqs, memory)
    assert lib.host_hip_pending() == 0
    return got


def visible(i, q_len, kv_len, prefix, window):
    """Positions in prefix ++ own keys that query i sees, as a half-open range."""
    n = prefix + kv_len
    last = i + n - q_len
    low = max(0, last - window + 1) if window else 0
    return (low, last + 1) if last + 1 > low else (0, 0)


def covered(got, seqs, heads, kv_heads, hd, window, prefix):
    """Every row's visible keys are in its parts exactly once, and every row is written exactly once."""
    group, wide = heads // kv_heads, 64 if hd > 256 else 128
    assert got.args["join_rows"] == max([j.n_rows for j in got.joins], default=0)
    part = {}  # partial row -> (q token, group row, first own key row, keys)
    assert got.args["prefix_len"] == prefix
    written, longest = {}, 0

    def keys(item, token):
        """The keys of the item that the row of this token sees, counted through the prefix."""
        i = token - item.q_token
        last = i + item.shift
        low = last - window + 1 if window else 0
        return max(low, item.k_lo), min(last + 1, item.k_hi)

    for it in got.items:
        assert 0 < it.n_rows <= (32 if it.narrow else wide) and it.k_lo <= it.k_hi
        longest = max(longest, it.k_hi - it.k_lo)
        for r in range(it.n_rows):
            row = it.row0 + r
            token = it.q_token + row // group
            lo, hi = keys(it, token)
            entry = (token, row % group, it.key0, lo, max(lo, hi))
            if it.part == DIRECT:
                assert (token, row % group) not in written
                written[token, row % group] = [entry]
            else:
                assert it.part + r not in part and it.part + r < got.args["part_rows"]
                part[it.part + r] = entry
    for j in got.joins:
        for r in range(j.n_rows):
            row = j.row0 + r
            name = (j.q_token + row // group, row % group)
            assert name not in written
            written[name] = []
            for side in range(2):
                for s in range(j.splits[side]):
                    e = part.pop(j.part[side] + s * j.stride[side] + r)
                    assert e[:2] == name
                    written[name].append(e)
    assert not part  # every partial row is read, once
    for q0, q_len, k0, kv_len in seqs:
        for i in range(q_len):
            lo, hi = visible(i, q_len, kv_len, prefix, window)
            for g in range(group):
                ranges = []
                for _, _, key0, a, b in written.pop((q0 + i, g)):
                    if b > a:
                        assert b <= prefix + kv_len and (b <= prefix or key0 == k0)
                        ranges.append((a, b))
                ranges.sort()
                for (_, b), (a, _) in zip(ranges, ranges[1:]):
                    assert a == b
                assert (ranges[0][0], ranges[-1][1]) == (lo, hi) if ranges else hi == lo
    assert not written
    assert len(got.joins) > 0 or all(it.part == DIRECT for it in got.items)


LAYOUTS = [(3, 1, 256), (4, 1, 512), (2, 1, 128), (32, 8, 128), (8, 8, 64), (40, 1, 64)]


@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("window", [0, 1, 37, 600])
def test_prompts_chunks_and_tokens(ctx, memory, heads, kv_heads, hd, window):
    cases = [[(0, 1, 0, 1)], [(0, 300, 0, 300)], [(0, 1, 0, 3001)], [(3, 7, 50, 9), (10, 0, 0, 5), (20, 40, 0, 1000)],
             [(0, 5, 10, 2), (5, 3, 0, 0), (8, 600, 7, 590)],  # queries before their first key
             [(i, 1, 17 * i, 1 + 61 * i) for i in range(40)]]
    for seqs in cases:
        covered(call(ctx, memory, seqs, heads, kv_heads, hd, window), seqs, heads, kv_heads, hd, window, 0)


@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("window", [0, 1, 50, 900])
def test_prefix(ctx, memory, heads, kv_heads, hd, window):
    cases = [[(0, 1, 0, 1)], [(0, 1, 0, 0), (1, 1, 0, 0)], [(0, 4, 0, 0)], [(0, 9, 0, 2), (9, 1, 3, 4)],
             [(i, 1, 7 * i, 1 + i % 5) for i in range(70)], [(0, 200, 0, 200), (200, 31, 900, 900), (300, 5, 40, 5)],
             [(0, 0, 0, 0), (0, 3, 2, 3), (3, 0, 0, 9), (3, 2, 0, 0), (5, 2, 1, 2)]]
    for seqs in cases:
        for prefix in (1, 130, 5000):
            got = call(ctx, memory, seqs, heads, kv_heads, hd, window, prefix)
            covered(got, seqs, heads, kv_heads, hd, window, prefix)


def test_a_batch_reads_its_prefix_once(ctx, memory):
    seqs = [(i, 1, 10 * i, 10) for i in range(32)]
    got = call(ctx, memory, seqs, 32, 8, 128, 0, 4096)
    shared = [it for it in got.items if it.k_lo < 4096]
    assert all(it.n_rows == 128 for it in shared) and sum(it.k_hi - it.k_lo for it in shared) == 4096


def test_a_short_prefix_needs_no_parts(ctx, memory):
    """Where fewer tiles over the prefix save less than the joins cost, each text takes prefix and own keys in one item."""
    for seqs, prefix in (([(i, 1, 10 * i, 10) for i in range(32)], 100), ([(60 * i, 60, 60 * i, 60) for i in range(32)], 400)):
        got = call(ctx, memory, seqs, 32, 8, 128, 0, prefix)
        assert not got.joins and all(it.part == DIRECT and it.k_lo == 0 and it.k_hi > prefix for it in got.items)


@pytest.mark.parametrize("seed", range(12))
def test_any_call(ctx, memory, seed):
    rng = random.Random(seed)
    heads, kv_heads, hd = rng.choice(LAYOUTS)
    prefix, window, seqs, q = rng.choice([0, 1, rng.randint(2, 3000)]), rng.choice([0, rng.randint(1, 700)]), [], 0
    for _ in range(rng.randint(1, 12)):
        q += rng.choice([0, 0, 0, rng.randint(1, 9)])
        n = rng.choice([0, 1, rng.randint(2, 90)])
        seqs.append((q, n, rng.randint(0, 500), rng.choice([0, n, n + rng.randint(0, 2000), rng.randint(0, 40)])))
        q += n
    covered(call(ctx, memory, seqs, heads, kv_heads, hd, window, prefix), seqs, heads, kv_heads, hd, window, prefix)


def test_nothing_to_do_launches_nothing(ctx, memory):
    for seqs in ([], [(0, 0, 0, 5)], [(4, 0, 0, 0), (4, 0, 0, 0)]):
        assert call(ctx, memory, seqs, 2, 1, 128, q_rows=4, kv_rows=9).names == []


def test_positions_past_32_bits_of_offsets(ctx, memory):
    """Key rows and strides whose byte offsets pass 2^32 reach the kernels as row numbers."""
    seqs = [(0, 1, (1 << 30) - 5000, 4000)]
    got = call(ctx, memory, seqs, 8, 1, 128, k_stride=1 << 24)
    covered(got, seqs, 8, 1, 128, 0, 0)
    assert got.args["k_stride"] == 1 << 24 and {it.key0 for it in got.items} == {(1 << 30) - 5000}


def test_scale(ctx, memory):
    """A negative scale flips q's signs, and a scale of 0 keeps hidden scores at -inf."""
    one = [(0, 1, 0, 1)]
    a = call(ctx, memory, one, 1, 1, 64, scale=-0.5).args
    assert a["q_flip"] == 0x80008000 and abs(a["c"] - 0.5 / np.log(2)) < 1e-6
    a = call(ctx, memory, one, 1, 1, 64, scale=0.0).args
    assert a["q_flip"] == 0 and a["c"] > 0


REFUSED = [dict(type=ge.GE_TYPE_F32), dict(hd=96), dict(hd=0), dict(heads=3, kv_heads=2), dict(heads=0), dict(kv_heads=0),
           dict(heads=8192, kv_heads=1), dict(window=-1), dict(window=1 << 30), dict(q_stride=100), dict(k_stride=132),
           dict(v_stride=-256), dict(out_stride=(1 << 24) + 8), dict(scale=float("inf")), dict(scale=float("nan")),
           dict(q_rows=-1), dict(kv_rows=-4), dict(q_rows=3), dict(kv_rows=8), dict(q_rows=1 << 30), dict(kv_rows=1 << 30),
           dict(seqs=[(0, 2, 0, 3), (1, 2, 0, 3)]), dict(seqs=[(2, 2, 0, 3), (0, 2, 0, 3)]),
           dict(seqs=[(0, 4, 0xffffffff, 2)]), dict(seqs=[(0xffffffff, 1, 0, 1)])]


@pytest.mark.parametrize("change", REFUSED, ids=str)
@pytest.mark.parametrize("prefix", [0, 7])
def test_refusals(ctx, memory, change, prefix):
    a = dict(seqs=[(0, 4, 0, 9)], heads=2, kv_heads=1, hd=128, q_rows=4, kv_rows=9)
    a.update(change)
    with pytest.raises(ge.GemmaEmbedError) as e:
        call(ctx, memory, a.pop("seqs"), a.pop("heads"), a.pop("kv_heads"), a.pop("hd"), prefix=prefix, **a)
    assert e.value.code == ge.GE_ERR_INVALID and "attention:" in e.value.message


def test_refused_pointers(ctx, memory):
    shape, seqs = ge.attention_shape(ge.GE_TYPE_F16, 2, 1, 128, 4, 9), [(0, 4, 0, 9)]
    good = [memory] * 4
    for i in range(4):
        for bad in (None, memory + 8):
            q, k, v, out = good[:i] + [bad] + good[i + 1:]
            with pytest.raises(ge.GemmaEmbedError):
                ctx.attention_causal(shape, q, k, v, seqs, out)
    for pk, pv in ((None, memory), (memory, None), (memory + 2, memory)):
        with pytest.raises(ge.GemmaEmbedError):
            ctx.attention_prefix(shape, memory, pk, pv, 5, memory, memory, seqs, memory)
    with pytest.raises(ge.GemmaEmbedError):
        ctx.attention_prefix(shape, memory, memory, memory, -1, memory, memory, seqs, memory)
    half = ge.attention_shape(ge.GE_TYPE_F16, 2, 1, 128, 4, 1 << 29)
    with pytest.raises(ge.GemmaEmbedError) as e:  # key rows and prefix together
        ctx.attention_prefix(half, memory, memory, memory, 1 << 29, memory, memory, seqs, memory)
    assert e.value.code == ge.GE_ERR_INVALID and "prefix together" in e.value.message
    assert lib.ge_op_attention_causal(ctx.handle, None, memory, memory, memory, None, 0, memory) == ge.GE_ERR_INVALID
    assert lib.ge_op_attention_causal(ctx.handle, C.byref(shape), memory, memory, memory, None, 1, memory) == ge.GE_ERR_INVALID
    assert lib.ge_op_attention_causal(None, C.byref(shape), memory, memory, memory, None, 0, memory) == ge.GE_ERR_INVALID
    # without own keys k and v may be null, and without a prefix its pointers
    ctx.attention_prefix(shape, memory, memory, memory, 5, None, None, [(0, 4, 0, 0)], memory)
    ctx.attention_prefix(shape, memory, None, None, 0, memory, memory, seqs, memory)


def test_a_failed_call_leaves_nothing_in_flight(ctx, memory):
    """The pinned lists and the partial rows are the next call's: a failing call has waited."""
    seqs = [(0, 1, 0, 9000)]
    for name in ("hipStreamSynchronize", "kernel:causal_kernel", "kernel:causal_join_kernel"):
        lib.host_hip_fail(name.encode(), 1)
        with pytest.raises(ge.GemmaEmbedError) as e:
            call(ctx, memory, seqs, 2, 1, 128)
        assert e.value.code == ge.GE_ERR_GPU
        assert lib.host_hip_pending() == 0
    covered(call(ctx, memory, seqs, 2, 1, 128), seqs, 2, 1, 128, 0, 0)
