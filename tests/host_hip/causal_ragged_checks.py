"""The plans of ragged batches, whose longest text is a large part of the work, on the host HIP runtime (host_hip.cpp).
Run by tests/test_causal_ragged_plan.py in a process of its own, whose GE_LIBRARY is the library's objects over that
runtime."""
import os
import sys

import pytest

import gemma_embed as ge

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from causal_checks import call, covered  # noqa: E402

CUS = 256


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def memory(ctx):
    return ctx.alloc(1 << 16)


def one_long(short, count, long):
    """Single tokens over `count` caches of `short` keys and one of `long`."""
    return [(i, 1, i * short, short) for i in range(count)] + [(count, 1, count * short, long)]


@pytest.mark.parametrize("heads,kv_heads,hd", [(32, 8, 128), (16, 16, 64), (4, 2, 256), (4, 1, 512)])
@pytest.mark.parametrize("count", [20, 127, 128, 700, 1100])
@pytest.mark.parametrize("prefix", [0, 30])
def test_one_long_text_among_short_ones(ctx, memory, heads, kv_heads, hd, count, prefix):
    """However many short texts stand beside it, the long one is split: no item takes longer than a CU's share of the
    call twice over."""
    seqs = one_long(100, count, 60000)
    got = call(ctx, memory, seqs, heads, kv_heads, hd, 0, prefix)
    covered(got, seqs, heads, kv_heads, hd, 0, prefix)
    total = sum(it.k_hi - it.k_lo for it in got.items) * kv_heads
    assert max(it.k_hi - it.k_lo for it in got.items) <= max(128, 2 * total // CUS + 64)


@pytest.mark.parametrize("heads,kv_heads,hd", [(32, 8, 128), (16, 16, 64)])
def test_a_long_prompt_among_short_ones(ctx, memory, heads, kv_heads, hd):
    seqs = [(10 * i, 10, 10 * i, 10) for i in range(200)] + [(2000, 40, 2000, 60000)]
    got = call(ctx, memory, seqs, heads, kv_heads, hd)
    covered(got, seqs, heads, kv_heads, hd, 0, 0)
    assert max(it.k_hi - it.k_lo for it in got.items) < 20000


@pytest.mark.parametrize("heads,kv_heads,hd", [(32, 8, 128), (16, 16, 64)])
def test_even_batches_are_not_split(ctx, memory, heads, kv_heads, hd):
    """Four items a CU and more whose longest is no more than a CU's share: nothing to even out."""
    for seqs in ([(i, 1, 900 * i, 500 + i % 400) for i in range(256)], [(0, 9000, 0, 9000)]):
        assert not call(ctx, memory, seqs, heads, kv_heads, hd).joins
