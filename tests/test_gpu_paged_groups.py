"""Attention over pages (ge_op_attention_paged) with many query heads to a KV head: single tokens then are wide items, and
none of their rows has hidden keys. Against float64, with the tolerances of test_gpu_paged.py."""
import numpy as np
import pytest

import gemma_embed as ge
from test_gpu_causal import BF16, F16, to_bits, to_float
from test_gpu_paged import INF, NAN, attend

pytestmark = pytest.mark.gpu
GROUPS = [(33, 1, 64), (48, 1, 128), (96, 2, 128), (40, 1, 256), (200, 1, 256), (48, 1, 512), (128, 1, 512)]
LENGTHS = [1, 8, 9, 31, 33, 40, 64, 65, 100, 129, 700]


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


def nan_in_page_0(q, cache):
    """No sequence has page 0, and neither do pools hold a number in it: what a group of keys past a sequence's end would
    read there is seen."""
    at = np.argwhere(cache.table == 0)
    if len(at):
        (slot, index), spare = at[0], next(p for p in range(1, cache.n_pages) if p not in cache.table)
        for pool in (cache.k, cache.v):
            pool[spare] = pool[0]
        cache.table[slot, index] = spare
        cache.ctx.page_table_set(cache.handle, [(slot, index, spare)])
    cache.k[0] = NAN[cache.kind]
    cache.v[0] = NAN[cache.kind]
    cache.v[0, 1::2] = INF[cache.kind]


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", GROUPS)
@pytest.mark.parametrize("page", [8, 32])
def test_tokens_past_whose_end_lies_nothing(ctx, heads, kv_heads, hd, kind, page):
    """Lengths off a block's multiple: the groups of 8 keys past the end are copied from resources of no bytes."""
    seqs = [(i, 1, m) for i, m in enumerate(LENGTHS)]
    attend(ctx, seqs, heads, kv_heads, hd, kind, page, seed=page, edit=nan_in_page_0)
    for m in (5, 42):  # alone, and in few parts
        attend(ctx, [(0, 1, m)], heads, kv_heads, hd, kind, page, seed=m, edit=nan_in_page_0)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", GROUPS)
def test_windows_and_caps_of_many_heads(ctx, heads, kv_heads, hd, kind):
    seqs = [(i, 1, m) for i, m in enumerate(LENGTHS)]
    attend(ctx, seqs, heads, kv_heads, hd, kind, 16, window=37, cap=20.0, seed=3, edit=nan_in_page_0)
    attend(ctx, seqs, heads, kv_heads, hd, kind, 16, cap=20.0, seed=4, edit=nan_in_page_0)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", GROUPS)
@pytest.mark.parametrize("window", [0, 50])
def test_chunks_of_many_heads(ctx, heads, kv_heads, hd, kind, window):
    """Stacked rows of a token in several tiles, and tiles that begin within a token."""
    attend(ctx, [(0, 3, 200), (3, 7, 7), (11, 2, 77), (13, 5, 2)], heads, kv_heads, hd, kind, 16, window=window, seed=5, edit=nan_in_page_0)


@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 1, 64), (4, 4, 128), (3, 1, 256), (2, 1, 512), (48, 1, 128)])
def test_infinite_values_of_keys_that_weigh_nothing(ctx, heads, kv_heads, hd):
    """A value that a row sees reaches it however little its key weighs, also where a whole part's scores fall past fp32's
    lowest: an infinity there is 0 times infinity in the definition."""
    def edit(q, cache):
        q[:] = to_bits(np.full(q.shape, 2.0 ** 40), BF16)
        for j in range(192):
            cache.row(cache.k, 0, j)[:] = to_bits(np.full((kv_heads, hd), -(2.0 ** 100)), BF16)
        cache.row(cache.v, 0, 5)[0, 3] = INF[BF16]
        cache.row(cache.v, 0, 70)[-1, hd - 1] = NAN[BF16]
        cache.row(cache.v, 0, 1500)[0, 9] = INF[BF16]

    got = attend(ctx, [(0, 1, 2000)], heads, kv_heads, hd, BF16, scale=2.0 ** -44, edit=edit, seed=hd)
    f = to_float(got[0], BF16).reshape(heads, hd)
    assert np.isnan(f[0, 3]) and np.isnan(f[-1, hd - 1]) and f[0, 9] == np.inf and np.isfinite(f[0, 4:9]).all()
