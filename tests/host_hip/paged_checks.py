"""A paged cache's entries on the host HIP runtime (host_hip.cpp): what they refuse, what a page table holds, and what
a call's launches are given. Run by tests/test_paged_host.py in a process of its own, whose GE_LIBRARY is the
library's objects over that runtime."""
import ctypes as C
import random
import re

import numpy as np
import pytest

import gemma_embed as ge

P, I, U = C.c_void_p, C.c_int, C.c_uint32
LAUNCH = C.CFUNCTYPE(None, C.c_char_p, C.POINTER(P))
lib = ge.lib
lib.host_hip_pending.restype = C.c_uint64
lib.host_hip_fail.argtypes = [C.c_char_p, I]
lib.host_hip_on_launch.argtypes = [LAUNCH]
F32, F16, BF16 = ge.GE_TYPE_F32, ge.GE_TYPE_F16, ge.GE_TYPE_BF16
DIRECT = 0xffffffff


class Item(C.Structure):
    """PagedItem, paged.hpp"""
    _fields_ = [(n, U) for n in ("q_token", "row0", "n_rows", "slot", "k_lo", "k_hi")] + \
        [("shift", C.c_int32)] + [(n, U) for n in ("part", "narrow", "next")]


class Join(C.Structure):
    """CausalJoin"""
    _fields_ = [(n, U) for n in ("q_token", "row0", "n_rows")] + [(n, U * 2) for n in ("part", "stride", "splits")]


class Args(C.Structure):
    """PagedArgs, paged.hpp: CausalArgs and the pages"""
    _fields_ = [(n, P) for n in ("q", "k", "v", "prefix_k", "prefix_v", "out")] + \
        [("unused", P), ("joins", C.POINTER(Join)), ("part_o", P), ("part_ml", P)] + \
        [(n, C.c_int64) for n in ("q_stride", "k_stride", "v_stride", "out_stride")] + [("part_rows", C.c_size_t)] + \
        [(n, I) for n in ("n_items", "n_joins", "join_rows", "group", "kv_heads", "window", "prefix_len")] + \
        [("c", C.c_float), ("q_flip", U), ("items", C.POINTER(Item)), ("table", P), ("page_stride", C.c_int64), ("slot_pages", I), ("page_shift", I),
         ("cap_z", C.c_float), ("cap_top", C.c_float)]


class JoinArgs(C.Structure):
    """CausalArgs"""
    _fields_ = Args._fields_[:Args._fields_.index(("items", C.POINTER(Item)))]


class JoinInline(C.Structure):
    """CausalInline, causal.hpp"""
    _fields_ = [("items", C.c_char * (48 * 36)), ("joins", Join * 40)]


class Append(C.Structure):
    """AppendItem, rotary.hpp"""
    _fields_ = [(n, U) for n in ("row0", "n", "slot", "first", "group0")]


class Heads(C.Structure):
    """HeadsArgs"""
    _fields_ = [(n, P) for n in ("q", "k", "v", "q_out", "k_out", "v_out", "q_norm", "k_norm", "positions", "turns", "table")] + \
        [("items", C.POINTER(Append))] + [(n, C.c_int64) for n in ("q_stride", "k_stride", "v_stride", "q_out_stride",
                                                                 "k_out_stride", "page_stride")] + \
        [(n, I) for n in ("heads", "kv_heads", "head_dim", "rows", "half", "pairs", "normed")] + \
        [(n, C.c_float) for n in ("eps", "fade", "gain")] + [(n, I) for n in ("rows_each", "workgroups", "n_items", "slot_pages", "page_shift")]


class Launches:
    """The launches of a block, by name, with copies of what they were given."""

    def __enter__(self):
        self.names, self.error, self.appended, self.items, self.joins, self.args, self.set = [], None, [], [], [], None, []

        def on_launch(name, args):
            try:
                name = name.decode()
                self.names.append(name)
                if "append_kernel" in name:
                    a, few = C.cast(args[0], C.POINTER(Heads))[0], C.cast(args[1], C.POINTER(Append * 160))[0]
                    self.args = {f: getattr(a, f) for f, _ in Heads._fields_ if f != "items"}
                    items, self.appended = [Append.from_buffer_copy((a.items or few)[i]) for i in range(a.n_items)], []
                    assert bool(a.items) == (a.n_items > 160) and (not a.items or a.workgroups == a.n_items)
                    for g in range(a.workgroups):  # what each takes
                        i = items[g] if a.items else [x for x in items if x.group0 <= g][-1]
                        skip = (g - i.group0) * a.rows_each
                        assert g >= i.group0 and skip < i.n
                        self.appended.append(Append(i.row0 + skip, min(i.n - skip, a.rows_each), i.slot, i.first + skip, g))
                elif "rotate_heads_kernel" in name:
                    a = C.cast(args[0], C.POINTER(Heads))[0]
                    self.args = {f: getattr(a, f) for f, _ in Heads._fields_ if f != "items"}
                elif "paged_kernel" in name:
                    a, few = C.cast(args[0], C.POINTER(Args))[0], C.cast(args[1], C.POINTER(Item * 90))[0]
                    self.args = {f: getattr(a, f) for f, _ in Args._fields_ if f not in ("items", "joins")}
                    self.chains = []  # of each workgroup
                    for at in range(a.n_items):
                        self.chains.append([])
                        while True:
                            self.chains[-1].append(Item.from_buffer_copy((a.items or few)[at]))
                            at = self.chains[-1][-1].next
                            if not at:
                                break
                            assert at >= a.n_items
                    self.items = [i for chain in self.chains for i in chain]
                elif "paged_join_kernel" in name:
                    a, few = C.cast(args[0], C.POINTER(JoinArgs))[0], C.cast(args[1], C.POINTER(JoinInline))[0]
                    self.joins = [Join.from_buffer_copy((a.joins or few.joins)[i]) for i in range(a.n_joins)]
                elif "table_set_kernel" in name:
                    n = C.cast(args[2], C.POINTER(I))[0]
                    e = C.cast(C.cast(args[1], C.POINTER(P))[0], C.POINTER(C.c_int32 * 2))
                    self.set = [tuple(e[i]) for i in range(n)]
            except BaseException as e:  # noqa: BLE001
                self.error = self.error or e
        self.callback = LAUNCH(on_launch)
        lib.host_hip_on_launch(self.callback)
        return self

    def __exit__(self, *exc):
        lib.host_hip_on_launch(LAUNCH())
        if self.error and not exc[0]:
            raise self.error


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def memory(ctx):
    return ctx.alloc(1 << 16)


@pytest.fixture
def table(ctx):
    """8 slots of 20 pages of 16 rows; slots 0 to 5 have 12 pages of their own each."""
    h = ctx.page_table_create(8, 20, 16, 100)
    ctx.page_table_set(h, [(s, i, 12 * s + i) for s in range(6) for i in range(12)])
    yield h
    ctx.page_table_destroy(h)


@pytest.fixture
def rotary(ctx):
    h = ctx.rotary_create(64, 1e4)
    yield h
    ctx.rotary_destroy(h)


def refused(call, *args, **kw):
    with pytest.raises(ge.GemmaEmbedError) as e:
        call(*args, **kw)
    assert e.value.code == ge.GE_ERR_INVALID and e.value.message
    assert lib.host_hip_pending() == 0


@pytest.mark.parametrize("bad", [dict(dims=0), dict(dims=-2), dict(dims=3), dict(dims=514), dict(layout=2), dict(layout=-1),
                                 dict(scaling=3), dict(scaling=-1), dict(base=0.0), dict(base=-1.0), dict(base=float("inf")),
                                 dict(base=float("nan")), dict(magnitude=float("nan")), dict(scaling=1, factor=0.0),
                                 dict(scaling=1, factor=float("inf")), dict(scaling=2, trained=0), dict(scaling=2, trained=-5),
                                 dict(scaling=2, trained=100, low_turns=4.0), dict(scaling=2, trained=100, high_turns=float("nan")),
                                 dict(scaling=2, trained=100, factor=-1.0)])
def test_refused_rotaries(ctx, bad):
    good = dict(dims=64, base=1e4)
    ctx.rotary_destroy(ctx.rotary_create(**good))
    refused(ctx.rotary_create, **dict(good, **bad))


def test_null_rotaries(ctx):
    h = P(1)
    assert lib.ge_op_rotary_create(ctx.handle, None, C.byref(h)) == ge.GE_ERR_INVALID and not h.value
    assert lib.ge_op_rotary_create(ctx.handle, C.byref(ge.ge_rotary_desc(2, base=1e4)), None) == ge.GE_ERR_INVALID
    assert lib.ge_op_rotary_destroy(ctx.handle, None) == ge.GE_OK


@pytest.mark.parametrize("bad", [(0, 4, 16, 10), (-1, 4, 16, 10), (4, 0, 16, 10), (4, 4, 16, 0), (4, 4, 0, 10), (4, 4, 4, 10), (4, 4, 24, 10),
                                 (4, 4, 2048, 10), (4, 4, -16, 10), (1 << 20, 1 << 10, 8, 10), (1, 1 << 27, 8, 10), (4, 4, 16, (1 << 28) + 1)])
def test_refused_tables(ctx, bad):
    refused(ctx.page_table_create, *bad)
    h = P(1)
    assert lib.ge_op_page_table_create(ctx.handle, *bad, C.byref(h)) == ge.GE_ERR_INVALID and not h.value


def test_failed_creations_leave_nothing(ctx):
    h = P(1)
    lib.host_hip_fail(b"hipMalloc", 1)
    assert lib.ge_op_page_table_create(ctx.handle, 2, 2, 16, 4, C.byref(h)) == ge.GE_ERR_GPU and not h.value
    for call in (b"hipMalloc", b"hipMemcpy"):
        lib.host_hip_fail(call, 1)
        assert lib.ge_op_rotary_create(ctx.handle, C.byref(ge.ge_rotary_desc(2, base=1e4)), C.byref(h)) == ge.GE_ERR_GPU and not h.value


@pytest.mark.parametrize("bad", [(8, 0, 1), (0, 20, 1), (0, 0, 100), (0, 0, -2)])
def test_refused_entries_change_nothing(ctx, table, bad):
    with Launches() as got:
        refused(ctx.page_table_set, table, [(0, 15, 99), bad])
    assert not got.names
    with Launches() as got:
        ctx.page_table_set(table, np.zeros((0, 3), np.int64))
    assert not got.names
    shape = ge.paged_shape(F16, 2, 1, 64, 1)
    refused(ctx.attention_paged, shape, 16, table, 16, 16, [(0, 1, 0, 16 * 12 + 1)], 16)


def test_entries_of_fractions_or_other_lengths(ctx, table):
    for bad in ([(0.5, 1, 1)], [(1, 2)], [1, 2, 3, 4], np.zeros((1, 1, 3), int)):
        with pytest.raises((TypeError, ValueError)):
            ctx.page_table_set(table, bad)
    with pytest.raises(OverflowError):
        ctx.page_table_set(table, [(0, 1 << 32, 0)])
    ctx.page_table_set(table, (0, 12, 90))


def test_the_later_of_two_entries_counts(ctx, table):
    with Launches() as got:
        ctx.page_table_set(table, [(6, 0, 80), (6, 1, 81), (6, 0, 82), (7, 0, 83), (7, 0, -1)])
    assert got.set == [(120, 82), (121, 81), (120, 82), (140, -1), (140, -1)]


def seen(ctx, table, slot, keys, q_len=1, window=0):
    shape = ge.paged_shape(F16, 2, 1, 64, q_len, window=window)
    try:
        ctx.attention_paged(shape, 16, table, 16, 16, [(0, q_len, slot, keys)], 16)
        return True
    except ge.GemmaEmbedError as e:
        assert e.code == ge.GE_ERR_INVALID
        return False


def test_pages_that_are_there(ctx, table):
    assert seen(ctx, table, 0, 192) and not seen(ctx, table, 0, 193) and not seen(ctx, table, 6, 1) and seen(ctx, table, 6, 0)
    ctx.page_table_set(table, [(0, 12, 90)])
    assert seen(ctx, table, 0, 208) and not seen(ctx, table, 0, 209)
    ctx.page_table_set(table, [(0, 14, 91)])  # a hole at 13
    assert seen(ctx, table, 0, 208) and not seen(ctx, table, 0, 209) and not seen(ctx, table, 0, 240)
    assert seen(ctx, table, 0, 240, window=16) and not seen(ctx, table, 0, 240, window=17)
    ctx.page_table_set(table, [(0, 13, 92)])
    assert seen(ctx, table, 0, 240)
    ctx.page_table_set(table, [(0, 0, -1), (0, 1, -1)])  # behind a window's reach
    assert not seen(ctx, table, 0, 240) and seen(ctx, table, 0, 240, window=208) and not seen(ctx, table, 0, 240, window=209)
    assert seen(ctx, table, 0, 240, q_len=100, window=109) and not seen(ctx, table, 0, 240, q_len=100, window=110)
    ctx.page_table_set(table, [(0, 14, -1)])
    assert not seen(ctx, table, 0, 240) and seen(ctx, table, 0, 224, window=5)
    ctx.page_table_set(table, [(0, i, -1) for i in range(20)])
    assert not seen(ctx, table, 0, 1)


def test_pages_against_a_plain_table(ctx):
    rng = random.Random(3)
    h = ctx.page_table_create(2, 12, 8, 30)
    plain = [[-1] * 12 for _ in range(2)]
    for _ in range(300):
        entries = [(rng.randrange(2), rng.randrange(12), rng.choice([-1, rng.randrange(30), rng.randrange(30)])) for _ in range(rng.randint(1, 4))]
        if rng.random() < 0.3:  # as a server does: the next page
            s = rng.randrange(2)
            used = [i for i in range(12) if plain[s][i] >= 0]
            at = used[-1] + 1 if used else 0
            entries = [(s, i, rng.randrange(30)) for i in range(at, min(12, at + rng.randint(1, 3)))] or entries
        ctx.page_table_set(h, entries)
        for s, i, page in entries:
            plain[s][i] = page
        for s in range(2):
            for keys in (1, 8, 9, 50, 96):
                assert seen(ctx, h, s, keys) == all(p >= 0 for p in plain[s][:(keys + 7) // 8])
                assert seen(ctx, h, s, keys, window=20) == all(p >= 0 for p in plain[s][max(0, keys - 20) // 8:(keys + 7) // 8])
    ctx.page_table_destroy(h)


@pytest.mark.parametrize("what", [b"kernel:table_set", b"hipStreamSynchronize"])
def test_a_set_that_fails_changes_nothing(ctx, table, what):
    lib.host_hip_fail(what, 1)
    with pytest.raises(ge.GemmaEmbedError) as e:
        ctx.page_table_set(table, [(0, 12, 90), (0, 0, -1), (0, 0, 7)])
    assert e.value.code == ge.GE_ERR_GPU
    ctx.page_table_set(table, [(1, 12, 91)])  # finds slot 1 only
    assert seen(ctx, table, 0, 192) and not seen(ctx, table, 0, 193) and seen(ctx, table, 1, 208)


# ---------------------------------------------------------------------------- rows of heads


ROTATE = dict(in_type=F16, type=F16, heads=4, kv_heads=2, head_dim=64, rows=3)


def rotate(ctx, memory, rotary, shape=None, **kw):
    a = dict(rotary=rotary, q=memory, k=memory, q_norm=None, k_norm=None, positions=memory, q_out=memory + 4096, k_out=memory + 4096)
    a.update(kw)
    ctx.rotate_heads(ge.heads_shape(**dict(ROTATE, **(shape or {}))), a["rotary"], a["q"], a["k"], a["q_norm"], a["k_norm"],
                     a["positions"], a["q_out"], a["k_out"])


@pytest.mark.parametrize("bad", [dict(type=F32), dict(type=ge.GE_TYPE_Q8_0), dict(in_type=BF16), dict(in_type=ge.GE_TYPE_Q8_0), dict(heads=-1),
                                 dict(kv_heads=-1), dict(heads=0, kv_heads=0), dict(heads=4097), dict(head_dim=0), dict(head_dim=33),
                                 dict(head_dim=514), dict(head_dim=62), dict(rows=-1), dict(rows=1 << 30), dict(normed=ge.GE_NORM_V),
                                 dict(normed=8), dict(normed=1, eps=-1.0), dict(normed=1, eps=float("nan")), dict(normed=1, eps=float("inf")),
                                 dict(q_stride=255), dict(k_stride=127), dict(q_out_stride=1), dict(k_out_stride=-128),
                                 dict(q_stride=(1 << 24) + 1)])
def test_refused_rows(ctx, memory, rotary, bad):
    rotate(ctx, memory, rotary)
    refused(rotate, ctx, memory, rotary, bad)


def test_refused_operands(ctx, memory, rotary):
    for bad in (dict(q=None), dict(k=None), dict(q_out=None), dict(k_out=None), dict(positions=None), dict(q=memory + 1), dict(k_out=memory + 1),
                dict(positions=memory + 2), dict(q_norm=memory + 2), dict(k_norm=memory + 1)):
        refused(rotate, ctx, memory, rotary, **bad)
    refused(rotate, ctx, memory, rotary, dict(in_type=F32), q=memory + 2)
    other = ge.Context.create(0)
    refused(rotate, other, memory, rotary)
    other.close()
    # nothing of what is not there
    rotate(ctx, memory, rotary, dict(heads=0), q=None, q_out=None)
    rotate(ctx, memory, rotary, dict(kv_heads=0), k=None, k_out=None)
    rotate(ctx, memory, None, positions=None)
    with Launches() as got:
        rotate(ctx, memory, rotary, dict(rows=0), q=None, k=None, q_out=None, k_out=None, positions=None)
    assert not got.names
    assert lib.ge_op_rotate_heads(ctx.handle, None, rotary, *[memory] * 7) == ge.GE_ERR_INVALID


def test_results_in_their_operands_place(ctx, memory, rotary, table):
    place = dict(q_out=memory, k_out=memory)
    seqs = [(0, 3, 0, 50)]
    rotate(ctx, memory, rotary, dict(q_stride=264, q_out_stride=264), **place)
    rotate(ctx, memory, rotary, dict(q_stride=264, rows=1), **place)
    append(ctx, memory, rotary, table, seqs, q_out=memory)
    for bad in (dict(q_stride=264), dict(k_stride=136), dict(k_out_stride=136), dict(in_type=F32), dict(in_type=F32, rows=1)):
        refused(rotate, ctx, memory, rotary, bad, **place)
    for bad in (dict(q_stride=264), dict(in_type=F32)):
        refused(append, ctx, memory, rotary, table, seqs, bad, q_out=memory)


def test_handles_end_in_their_context(ctx):
    rotary, table = ctx.rotary_create(64, 1e4), ctx.page_table_create(1, 1, 8, 1)
    other = ge.Context.create(0)
    refused(other.rotary_destroy, rotary)
    refused(other.page_table_destroy, table)
    assert lib.ge_op_rotary_destroy(None, rotary) == lib.ge_op_page_table_destroy(None, table) == ge.GE_ERR_INVALID
    other.close()
    ctx.page_table_set(table, [(0, 0, 0)])  # still there
    ctx.rotary_destroy(rotary)
    ctx.page_table_destroy(table)
    ctx.rotary_destroy(None)
    ctx.page_table_destroy(None)


def unit_of(name):
    return int(re.search(r"Li(\d)EEEv", name).group(1))


@pytest.mark.parametrize("shape,kw,unit", [
    ({}, {}, 8), (dict(head_dim=80), {}, 8), (dict(in_type=F32), {}, 8), (dict(q_stride=264), {}, 8), (dict(q_stride=260), {}, 4),
    (dict(q_stride=258), {}, 2), (dict(q_stride=257), {}, 1), (dict(in_type=F32, q_stride=260), {}, 8), (dict(in_type=F32, k_stride=130), {}, 2),
    (dict(in_type=F32, k_stride=129), {}, 1), (dict(k_out_stride=132), {}, 4), (dict(q_out_stride=262), {}, 2),
    (dict(head_dim=72), {}, 4), (dict(head_dim=68), {}, 2), (dict(head_dim=66), {}, 1), (dict(head_dim=260), {}, 1), (dict(head_dim=264), {}, 4),
    ({}, dict(q=2), 1), ({}, dict(q=4), 2), ({}, dict(k_out=8), 4), (dict(in_type=F32), dict(k=8), 2), (dict(in_type=F32), dict(k=4), 1),
    (dict(in_type=F32), dict(k=16), 8), ({}, dict(q_norm=4), 8), ({}, dict(positions=4), 8)])
def test_units(ctx, memory, rotary, shape, kw, unit):
    """Elements move in the largest units that every address, stride and part allows."""
    with Launches() as got:
        rotate(ctx, memory, rotary, shape, **{n: memory + (4096 if n.endswith("out") else 0) + x for n, x in kw.items()})
    assert len(got.names) == 1 and unit_of(got.names[0]) == unit


def test_parts_of_a_head(ctx, memory):
    for dims, unit in ((16, 8), (48, 8), (24, 4), (20, 2), (36, 2), (2, 1), (34, 1), (64, 8)):
        h = ctx.rotary_create(dims, 1e4)
        with Launches() as got:
            rotate(ctx, memory, h)
        assert unit_of(got.names[0]) == unit and got.args["half"] == dims // 2
        ctx.rotary_destroy(h)
    h = ctx.rotary_create(4, 1e4)  # more units of 2 than lanes
    for hd, unit in ((256, 2), (512, 1)):
        with Launches() as got:
            rotate(ctx, memory, h, dict(head_dim=hd))
        assert unit_of(got.names[0]) == unit
    ctx.rotary_destroy(h)


def test_magnitudes(ctx, memory):
    for m, fade, gain in ((0.0, 1.0, 1.0), (1.0, 1.0, 1.0), (0.5, 0.5, 1.0), (1.25, 1.0, 1.25), (-2.0, 1.0, -2.0), (-0.5, -0.5, 1.0)):
        h = ctx.rotary_create(64, 1e4, magnitude=m)
        with Launches() as got:
            rotate(ctx, memory, h)
        assert (got.args["fade"], got.args["gain"]) == (fade, gain)
        ctx.rotary_destroy(h)


@pytest.mark.parametrize("scaling,trained,factor", [(0, 0, 8.0), (1, 0, 8.0), (2, 8192, 8.0), (2, 100, 0.5)])
@pytest.mark.parametrize("dims", [2, 64, 128])
def test_frequencies(ctx, memory, dims, scaling, trained, factor):
    """Turns a position, as the definition has them (float64's rounding of a few products)."""
    h = ctx.rotary_create(dims, 5e5, scaling=scaling, factor=factor, trained=trained)
    with Launches() as got:
        rotate(ctx, memory, h, dict(head_dim=128))
    f = np.float64(np.float32(5e5)) ** (-2.0 * np.arange(dims // 2) / dims)
    w = np.clip((trained * f / (2 * np.pi) - 1.0) / 3.0, 0.0, 1.0)
    want = [f, f / factor, f * (w + (1 - w) / factor)][scaling] / (2 * np.pi)
    turns = np.ctypeslib.as_array(C.cast(got.args["turns"], C.POINTER(C.c_double)), (dims // 2,))
    np.testing.assert_allclose(turns, want, rtol=1e-14)
    ctx.rotary_destroy(h)


# ---------------------------------------------------------------------------- appending


def append(ctx, memory, rotary, table, seqs, shape=None, **kw):
    a = dict(rotary=rotary, q=memory, k=memory, v=memory, q_norm=None, k_norm=None, positions=None, q_out=memory + 4096, k_pages=memory,
             v_pages=memory)
    a.update(kw)
    ctx.paged_append(ge.heads_shape(**dict(dict(ROTATE, rows=500), **(shape or {}))), a["rotary"], a["q"], a["k"], a["v"], a["q_norm"], a["k_norm"],
                     a["positions"], table, seqs, a["q_out"], a["k_pages"], a["v_pages"])


def test_refused_appends(ctx, memory, rotary, table):
    good = [(0, 3, 0, 50), (3, 1, 1, 1)]
    append(ctx, memory, rotary, table, good)
    append(ctx, memory, rotary, table, good, dict(normed=7))
    for shape in (dict(kv_heads=0), dict(v_stride=127), dict(page_stride=2047), dict(page_stride=2052), dict(page_stride=-8), dict(normed=8),
                  dict(page_stride=(1 << 40) + 8)):
        refused(append, ctx, memory, rotary, table, good, shape)
    append(ctx, memory, rotary, table, good, dict(k_out_stride=1 << 60, page_stride=2056))  # not an operand of this call
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(k_pages=None), dict(v_pages=None), dict(positions=memory + 1),
                dict(v=memory + 1), dict(k_pages=memory + 1)):
        refused(append, ctx, memory, rotary, table, good, **bad)
    append(ctx, memory, rotary, table, good, dict(heads=0), q=None, q_out=None)
    for seqs in ([(0, 3, 8, 50)], [(0, 3, 6, 50)], [(0, 3, 0, 2)], [(0, 3, 0, 193)], [(498, 3, 0, 50)], [(0, 3, 0, 50), (2, 1, 1, 5)],
                 [(5, 1, 0, 5), (0, 1, 1, 5)], [(0, 3, 0, 321)], [(0xffffffff, 2, 0, 50)]):
        refused(append, ctx, memory, rotary, table, seqs)
    refused(append, ctx, memory, rotary, None, good)
    other = ge.Context.create(0)
    refused(append, other, memory, None, table, good)
    other.close()
    with Launches() as got:
        append(ctx, memory, rotary, table, [], k=None)
        append(ctx, memory, rotary, table, [(3, 0, 0, 0), (1, 0, 7, 9)], k=None)
    assert not got.names


def test_a_page_has_one_writer(ctx, memory, rotary, table):
    ctx.page_table_set(table, [(6, 0, 0), (6, 1, 80), (6, 2, 80), (7, 0, 0), (7, 1, 81)])
    append(ctx, memory, rotary, table, [(0, 1, 0, 1)])
    append(ctx, memory, rotary, table, [(0, 1, 6, 1)])  # the same page in another call
    refused(append, ctx, memory, rotary, table, [(0, 1, 0, 1), (1, 1, 6, 2)])   # page 0 twice
    refused(append, ctx, memory, rotary, table, [(0, 1, 0, 50), (1, 1, 0, 50)])  # one slot twice
    refused(append, ctx, memory, rotary, table, [(0, 17, 6, 33 + 15)])  # page 80 at two places
    append(ctx, memory, rotary, table, [(0, 10, 6, 26)])
    append(ctx, memory, rotary, table, [(0, 1, 6, 17), (1, 1, 7, 17)])  # slots that share page 0, each writing a page of its own
    append(ctx, memory, rotary, table, [(0, 16, 0, 16), (16, 16, 0, 32), (32, 5, 0, 37)])  # one slot's pages by turns


@pytest.mark.parametrize("seqs", [[(0, 1, 0, 1)], [(0, 192, 0, 192)], [(3, 5, 2, 20), (8, 0, 1, 3), (8, 37, 1, 100), (60, 1, 4, 17)],
                                  [(5 * i, 1 + i % 3, i, 3 + 17 * i) for i in range(6)]])
def test_rows_of_an_append(ctx, memory, rotary, table, seqs):
    with Launches() as got:
        append(ctx, memory, rotary, table, seqs)
    rows = [(i.row0 + r, i.slot, i.first + r) for i in got.appended for r in range(i.n)]
    assert sorted(rows) == sorted((q + r, s, m - n + r) for q, n, s, m in seqs for r in range(n))
    a = got.args
    assert (a["slot_pages"], a["page_shift"], a["page_stride"]) == (20, 4, 16 * 2 * 64) and all(i.n <= 4 for i in got.appended)
    assert lib.host_hip_pending() == 0


def test_rows_of_a_long_append(ctx, memory):
    h = ctx.page_table_create(400, 8, 1024, 400 * 8)
    ctx.page_table_set(h, [(s, i, 8 * s + i) for s in range(400) for i in range(8)])
    for seqs in ([(0, 8192, 3, 8192)], [(i, 1, i, 1 + i) for i in range(400)], [(100 * i, 97, i, 1000) for i in range(200)],
                 [(8000 * i, 8000, i, 8191) for i in range(10)]):
        with Launches() as got:
            append(ctx, memory, None, h, seqs, dict(rows=1 << 17) if len(seqs) != 10 else dict(rows=80000))
        rows = [(i.row0 + r, i.slot, i.first + r) for i in got.appended for r in range(i.n)]
        assert sorted(rows) == sorted((q + r, s, m - n + r) for q, n, s, m in seqs for r in range(n))
        assert len(got.appended) <= 5120 + len(seqs)
    ctx.page_table_destroy(h)


# ---------------------------------------------------------------------------- attention


def attend(ctx, memory, table, seqs, heads=4, kv_heads=2, hd=64, **kw):
    names = {n: kw.pop(n) for n in list(kw) if n in ("q", "k_pages", "v_pages", "out")}
    a = dict(dict(q=memory, k_pages=memory, v_pages=memory, out=memory), **names)
    shape = ge.paged_shape(kw.pop("type", F16), heads, kv_heads, hd, kw.pop("q_rows", 2000), **kw)
    with Launches() as got:
        ctx.attention_paged(shape, a["q"], table, a["k_pages"], a["v_pages"], seqs, a["out"])
    assert lib.host_hip_pending() == 0
    return got


def test_refused_attention(ctx, memory, table):
    good = [(0, 3, 0, 50), (3, 1, 1, 100)]
    attend(ctx, memory, table, good)
    nan, inf = float("nan"), float("inf")
    for bad in (dict(type=F32), dict(hd=80), dict(hd=0), dict(heads=3), dict(heads=0), dict(kv_heads=0), dict(heads=4098), dict(q_rows=-1),
                dict(q_rows=1 << 30), dict(window=-1), dict(window=1 << 30), dict(scale=nan), dict(scale=inf), dict(cap=nan), dict(cap=inf),
                dict(cap=-1.0), dict(cap=3e38), dict(cap=1025.0), dict(cap=30000.0), dict(q_stride=255), dict(q_stride=260), dict(out_stride=8), dict(page_stride=2047), dict(page_stride=100),
                dict(q=None), dict(out=None), dict(k_pages=None), dict(v_pages=None), dict(q=memory + 8), dict(out=memory + 2),
                dict(k_pages=memory + 8), dict(q_rows=1 << 29, heads=8, kv_heads=1)):
        refused(attend, ctx, memory, table, good, **bad)
    for seqs in ([(0, 1, 8, 1)], [(0, 1, 6, 1)], [(0, 1, 0, 193)], [(0, 1, 0, 400)], [(1999, 2, 0, 5)], [(0, 3, 0, 50), (2, 1, 1, 5)]):
        refused(attend, ctx, memory, table, seqs)
    refused(attend, ctx, memory, None, good)
    other = ge.Context.create(0)
    refused(attend, other, memory, table, good)
    other.close()
    assert not attend(ctx, memory, table, [], q=None).names
    assert not attend(ctx, memory, table, [(0, 0, 0, 50)], q=None).names
    attend(ctx, memory, table, [(0, 5, 7, 0)], k_pages=None, v_pages=None)  # rows that see nothing


def covered(got, seqs, heads, kv_heads, hd, window):
    """Every row's visible keys are in its parts exactly once, every row is written exactly once, and an item's keys
    begin at a multiple of 8."""
    group, parts, written = heads // kv_heads, {}, {}
    slots = {q + i: (s, m - n) for q, n, s, m in seqs for i in range(n)}
    first = {q + i: q for q, n, _, _ in seqs for i in range(n)}
    for it in got.items:
        assert it.k_lo % 8 == 0 and it.k_lo <= it.k_hi and (it.n_rows <= 32) == bool(it.narrow)
        for r in range(it.row0, it.row0 + it.n_rows):
            token = it.q_token + r // group
            slot, shift = slots[token]
            assert (it.slot, it.shift) == (slot, shift)
            last = r // group + shift
            keys = set(range(max(it.k_lo, last - window + 1 if window else 0), min(it.k_hi, last + 1)))
            if it.part == DIRECT:
                assert (token, r % group) not in written
                written[token, r % group] = keys
            else:
                assert it.part + r - it.row0 not in parts
                parts[it.part + r - it.row0] = (token, r % group, keys)
    for j in got.joins:
        for r in range(j.n_rows):
            token, head = j.q_token + (j.row0 + r) // group, (j.row0 + r) % group
            keys = set()
            assert j.splits[1] == 0
            for s in range(j.splits[0]):
                t, h, more = parts.pop(j.part[0] + s * j.stride[0] + r)
                assert (t, h) == (token, head) and not keys & more
                keys |= more
            assert (token, head) not in written
            written[token, head] = keys
    assert not parts and (got.joins or not got.args["n_joins"])
    at_once = {64: 768, 128: 512, 256: 512, 512: 256}[hd] // kv_heads
    if got.joins:  # equal shares: no more workgroups than run at once
        assert len(got.chains) <= max(at_once, 1024 // kv_heads)
    for token, (_, shift) in slots.items():
        last = token - first[token] + shift
        for h in range(group):
            assert written.pop((token, h)) == set(range(max(0, last - window + 1 if window else 0), last + 1))
    assert not written


@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 1, 64), (6, 2, 128), (3, 1, 256), (2, 1, 512)])
@pytest.mark.parametrize("window", [0, 1, 7, 100, 1500])
def test_the_plan_covers_every_key_once(ctx, memory, heads, kv_heads, hd, window):
    h = ctx.page_table_create(100, 600, 8, 600)
    ctx.page_table_set(h, [(s, i, i) for s in range(100) for i in range(600)])
    for seqs in ([(0, 1, 0, 1)], [(0, 1, 3, 4800)], [(0, 300, 2, 300)], [(0, 1500, 2, 4700)], [(0, 200, 1, 4001), (200, 1, 5, 4800), (205, 9, 7, 4)],
                 [(i, 1, i, 1 + 48 * i) for i in range(100)], [(0, 3, 0, 0), (3, 50, 9, 20)]):
        got = attend(ctx, memory, h, seqs, heads, kv_heads, hd, window=window)
        covered(got, seqs, heads, kv_heads, hd, window)
        a = got.args
        assert (a["slot_pages"], a["page_shift"], a["page_stride"], a["group"]) == (600, 3, 8 * kv_heads * hd, heads // kv_heads)
    ctx.page_table_destroy(h)


@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 1, 64), (1024, 1024, 64), (4, 1, 512)])
@pytest.mark.parametrize("window", [0, 300000])
def test_the_plan_of_long_caches(ctx, memory, heads, kv_heads, hd, window):
    h = ctx.page_table_create(3, 600, 1024, 600)
    ctx.page_table_set(h, [(s, i, i) for s in range(3) for i in range(600)])
    for seqs in ([(0, 1, 0, 614400)], [(0, 2, 0, 600001), (2, 1, 1, 100), (3, 1, 2, 345678)]):
        got = attend(ctx, memory, h, seqs, heads, kv_heads, hd, window=window)
        covered(got, seqs, heads, kv_heads, hd, window)
        if kv_heads > 1000:  # whole tiles, the longest first
            units = [-(-(i.k_hi - i.k_lo) // 64) for i in got.items]
            assert units == sorted(units, reverse=True) and not got.joins
    ctx.page_table_destroy(h)


@pytest.mark.parametrize("n", [33, 300, 1500])
def test_the_longest_tiles_come_first(ctx, memory, n):
    """Items of one kind of workgroup each, sorted; equal ones in the sequences' order."""
    h = ctx.page_table_create(n, 4, 64, 4)
    ctx.page_table_set(h, [(s, i, i) for s in range(n) for i in range(4)])
    seqs = [(i, 1, i, 1 + 7 * i % 128) for i in range(n)]
    got = attend(ctx, memory, h, seqs, q_rows=n)
    covered(got, seqs, 4, 2, 64, 0)
    order = [(-(-(i.k_hi - i.k_lo) // 64), i.slot) for i in got.items]
    assert order == sorted(order, key=lambda x: (-x[0], x[1])) and not got.joins
    ctx.page_table_destroy(h)


def test_caps(ctx, memory, table):
    seqs = [(0, 1, 0, 50)]
    a = attend(ctx, memory, table, seqs, scale=-0.5).args
    assert a["cap_top"] == 0 and a["q_flip"] == 0x80008000 and a["c"] == pytest.approx(0.5 * 1.4426950408889634)
    a = attend(ctx, memory, table, seqs, scale=-0.5, cap=50.0).args
    assert a["c"] == 1.0 and a["cap_z"] == pytest.approx(0.02 * 1.4426950408889634) and a["cap_top"] == pytest.approx(50 * 1.4426950408889634)
    assert a["q_flip"] == 0x80008000
    a = attend(ctx, memory, table, seqs, scale=3e38, cap=1e-30).args
    assert np.isfinite(a["cap_z"]) and a["cap_top"] > 0


@pytest.mark.parametrize("what", [b"kernel:paged_kernel", b"kernel:paged_join", b"hipStreamSynchronize", b"hipMalloc"])
def test_a_call_that_fails_leaves_nothing_in_flight(ctx, memory, what):
    h = ctx.page_table_create(1, 5000, 16, 5000)
    ctx.page_table_set(h, [(0, i, i) for i in range(5000)])
    c = ge.Context.create(0)  # with no temporaries yet
    own = c.page_table_create(1, 5000, 16, 5000)
    c.page_table_set(own, [(0, i, i) for i in range(5000)])
    lib.host_hip_fail(what, 1)
    with pytest.raises(ge.GemmaEmbedError) as e:
        attend(c, memory, own, [(0, 1, 0, 80000)])
    assert e.value.code == ge.GE_ERR_GPU
    assert lib.host_hip_pending() == 0
    attend(c, memory, own, [(0, 1, 0, 80000)])
    c.page_table_destroy(own)
    c.close()
    ctx.page_table_destroy(h)
