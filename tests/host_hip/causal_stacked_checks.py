"""The plans of calls over a shared prefix whose texts stack up (tests/causal_stacked.py), on the host HIP runtime
(host_hip.cpp). Run by tests/test_causal_stacked_plan.py in a process of its own, whose GE_LIBRARY is the
library's objects over that runtime."""
import os
import sys

import pytest

import gemma_embed as ge

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from causal_checks import call, covered  # noqa: E402
from causal_stacked import STACKED  # noqa: E402

ALL = 1 << 30  # the shift of an item whose rows all see its keys


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def memory(ctx):
    return ctx.alloc(1 << 16)


@pytest.mark.parametrize("name,heads,kv_heads,hd,prefix,seqs", STACKED, ids=[f"{c[0]}-{c[1]}-{c[2]}-{c[3]}" for c in STACKED])
def test_the_texts_stack(ctx, memory, name, heads, kv_heads, hd, prefix, seqs):
    got = call(ctx, memory, seqs, heads, kv_heads, hd, 0, prefix)
    covered(got, seqs, heads, kv_heads, hd, 0, prefix)
    stacked = [it for it in got.items if it.shift == ALL]
    assert stacked and all(it.k_hi <= prefix for it in stacked)
    rows = sum(n for _, n, _, _ in seqs if n) * (heads // kv_heads)
    assert sum(it.n_rows for it in stacked if it.k_lo == 0) > rows // 2
    if name == "alone":
        assert not any(j.splits[0] for j in got.joins)
    else:
        assert any(j.splits[0] and j.splits[1] for j in got.joins)
    if name == "split":
        assert any(j.splits[1] > 1 for j in got.joins)
    if name == "apart":
        assert any(it.shift != ALL and it.k_lo < prefix for it in got.items)
