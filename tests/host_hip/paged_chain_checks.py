"""The plans of paged_chains.py's calls on the host HIP runtime (host_hip.cpp): that they do chain items and pass a launch's
joins. Run by tests/test_paged_chains_host.py in a process of its own, whose GE_LIBRARY is the library's objects over
that runtime."""
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import paged_chains  # noqa: E402
from paged_checks import attend, covered, ctx, memory  # noqa: E402, F401 (fixtures)

INLINE_ITEMS, INLINE_JOINS = 90, 40  # kPagedInlineItems, kCausalInlineJoins


@pytest.fixture(scope="module")
def table(ctx):  # noqa: F811
    h = ctx.page_table_create(100, 125, 8, 125)
    ctx.page_table_set(h, [(s, i, i) for s in range(100) for i in range(125)])
    yield h
    ctx.page_table_destroy(h)


def planned(ctx, memory, table, seqs, heads, kv_heads, hd, window):  # noqa: F811
    call = [(q, n, i, m) for i, (q, n, m) in enumerate(seqs)]
    got = attend(ctx, memory, table, call, heads, kv_heads, hd, window=window)
    covered(got, call, heads, kv_heads, hd, window)
    return got


@pytest.mark.parametrize("heads,kv_heads,hd", paged_chains.LAYOUTS)
@pytest.mark.parametrize("call", paged_chains.CALLS)
@pytest.mark.parametrize("window", [0, paged_chains.WINDOW])
def test_items_follow_each_other(ctx, memory, table, heads, kv_heads, hd, call, window):  # noqa: F811
    got = planned(ctx, memory, table, paged_chains.CALLS[call], heads, kv_heads, hd, window)
    assert len(got.chains) <= 8 and max(map(len, got.chains)) >= 4
    assert (len(got.items) > INLINE_ITEMS) == (call == "a list of items")
    kinds = [[bool(i.narrow) for i in chain] for chain in got.chains]
    if call == "tokens":
        assert all(all(k) for k in kinds)
    else:  # a wide item behind a narrow one, and a narrow one behind a wide one
        pairs = {p for k in kinds for p in zip(k, k[1:])}
        assert {(True, False), (False, True)} <= pairs


@pytest.mark.parametrize("heads,kv_heads,hd", paged_chains.JOINED)
def test_more_joins_than_a_launchs_arguments_hold(ctx, memory, table, heads, kv_heads, hd):  # noqa: F811
    got = planned(ctx, memory, table, paged_chains.joined(), heads, kv_heads, hd, 0)
    assert len(got.joins) > INLINE_JOINS


AT_ONCE = {64: 1024, 128: 512, 256: 512, 512: 256}  # workgroups on the GPU: 256 CUs of paged_workgroups


@pytest.fixture(scope="module")
def long_table(ctx):  # noqa: F811
    h = ctx.page_table_create(8, 1024, 64, 1024)
    ctx.page_table_set(h, [(s, i, i) for s in range(8) for i in range(1024)])
    yield h
    ctx.page_table_destroy(h)


LONG = [[(0, 1, 9000)], [(0, 1, 12000)], [(0, 1, 16319)], [(0, 1, 16320)], [(0, 1, 24000)], [(0, 1, 32000)], [(0, 1, 65536)],
        [(0, 1, 30000), (1, 1, 9000), (2, 1, 100)], [(i, 1, 8000 + 4000 * i) for i in range(8)], [(0, 150, 30000)], [(0, 200, 60000)],
        [(0, 150, 12000), (150, 150, 60000)], [(0, 1500, 4700)], [(0, 700, 2500), (700, 300, 9000), (1000, 1, 40)]]


@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 1, 64), (16, 8, 64), (6, 2, 128), (3, 1, 256), (2, 1, 512), (8, 8, 512)])
@pytest.mark.parametrize("seqs", LONG)
def test_workgroups_and_parts_of_a_row(ctx, memory, long_table, heads, kv_heads, hd, seqs):  # noqa: F811
    """Single tokens are cut into shares, one for each workgroup that runs at once at most, a row into 255 and a border; tiles of
    chunks into parts that fill two rounds at most."""
    got = attend(ctx, memory, long_table, [(q, n, i, m) for i, (q, n, m) in enumerate(seqs)], heads, kv_heads, hd)
    group, wide = heads // kv_heads, 128 if hd <= 256 else 64  # paged_wide_rows
    tiles = sum(-(-n * group // wide) for _, n, _ in seqs)
    if not got.joins:
        return
    if 2 * len(seqs) > tiles or len(got.items) > len(got.chains):
        assert len(got.chains) <= AT_ONCE[hd] // kv_heads
        assert max(j.splits[0] for j in got.joins) <= 256
    else:
        assert len(got.chains) <= 2 * AT_ONCE[hd] // kv_heads
