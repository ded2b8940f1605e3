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
