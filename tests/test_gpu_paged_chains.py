"""Attention over pages (ge_op_attention_paged) where workgroups take several items one after another over the same LDS, and
where a launch's items and joins are lists in memory (paged_chains.py, whose plans the host checks look at). Against
float64, with the tolerances of test_gpu_paged.py."""
import numpy as np
import pytest

import paged_chains
import test_gpu_paged
from test_gpu_causal import BF16, F16, to_bits, to_float

pytestmark = pytest.mark.gpu
COMMON = 24  # pages that all slots share


@pytest.fixture(scope="module")
def ctx():
    import gemma_embed as ge
    c = ge.Context.create(0)
    yield c
    c.close()


class Shared:
    """test_gpu_paged's Cache for long lists of sequences: pages of 16 keys, all but a slot's last one out of a few that
    slots share. Past a sequence's end its last page holds NaN."""

    def __init__(self, ctx, rng, lengths, page, kv_heads, hd, kind, gap=0, values=1.0):
        assert page == 16 and not gap
        self.ctx, self.page, self.kind, self.kv_heads, self.hd = ctx, page, kind, kv_heads, hd
        self.elements = self.stride = page * kv_heads * hd
        self.n_pages = COMMON + len(lengths) + 1
        counts = [-(-n // page) for n in lengths]
        self.table = np.full((len(lengths), max(counts)), -1, np.int64)
        self.k, self.v = (to_bits(rng.standard_normal((self.n_pages, self.elements)), kind) for _ in range(2))
        for s, n in enumerate(lengths):
            if n:
                self.table[s, :counts[s]] = np.append(rng.integers(0, COMMON, counts[s] - 1), COMMON + s)
            for pool in (self.k, self.v):
                self.heads(pool)[COMMON + s, :, (n - 1) % page + 1 if n else 0:] = test_gpu_paged.NAN[kind]
        self.handle = ctx.page_table_create(*self.table.shape, page, self.n_pages)
        slots, index = np.nonzero(self.table >= 0)
        ctx.page_table_set(self.handle, np.stack([slots, index, self.table[slots, index]], 1))

    def heads(self, pool):
        return pool.reshape(self.n_pages, self.kv_heads, self.page, self.hd)

    def rows(self, pool, slot, first, end):
        pages = self.heads(pool)[self.table[slot, :-(-end // self.page)]]
        return to_float(pages.transpose(0, 2, 1, 3).reshape(-1, self.kv_heads, self.hd)[first:end], self.kind)

    def close(self):
        self.ctx.page_table_destroy(self.handle)


@pytest.fixture(autouse=True)
def shared_pages(monkeypatch):
    monkeypatch.setattr(test_gpu_paged, "Cache", Shared)


# every head dim with and without a window and a cap
FORMS = [(0, 0.0), (paged_chains.WINDOW, 20.0)]
CASES = [(*x, (F16, BF16)[i % 2], *FORMS[i % 2]) for i, x in enumerate(paged_chains.LAYOUTS)] + [(64, 64, 256, BF16, *FORMS[1])]


@pytest.mark.parametrize("heads,kv_heads,hd,kind,window,cap", CASES)
@pytest.mark.parametrize("call", paged_chains.CALLS)
def test_items_one_after_another(ctx, heads, kv_heads, hd, kind, call, window, cap):
    test_gpu_paged.attend(ctx, paged_chains.CALLS[call], heads, kv_heads, hd, kind, window=window, cap=cap, seed=hd)


@pytest.mark.parametrize("heads,kv_heads,hd,kind", [(*paged_chains.LAYOUTS[i], k) for i, k in ((0, BF16), (2, F16), (4, BF16), (6, F16))])
@pytest.mark.parametrize("window", [0, paged_chains.WINDOW])
def test_infinite_values_among_them(ctx, heads, kv_heads, hd, kind, window):
    """Values that only some of a chunk's rows see, held back and added to what the item has stored, between items that
    hold nothing back."""
    seqs = paged_chains.CALLS["chunks among them"]

    def edit(q, cache):
        v = cache.heads(cache.v)
        for s, (_, n, m) in enumerate(seqs):
            if n > 1 and m % 16 > 2:  # its last two keys
                v[COMMON + s, 0, (m - 1) % 16, 1] = test_gpu_paged.INF[kind]
                v[COMMON + s, -1, (m - 2) % 16, hd - 1] = test_gpu_paged.NAN[kind]
    test_gpu_paged.attend(ctx, seqs, heads, kv_heads, hd, kind, window=window, seed=hd, edit=edit)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", paged_chains.JOINED)
def test_lists_of_joins(ctx, heads, kv_heads, hd, kind):
    test_gpu_paged.attend(ctx, paged_chains.joined(), heads, kv_heads, hd, kind, seed=hd)
    test_gpu_paged.attend(ctx, paged_chains.joined(), heads, kv_heads, hd, kind, cap=20.0, seed=hd + 1)


def test_the_same_bits_every_time(ctx):
    a, b = (test_gpu_paged.attend(ctx, paged_chains.CALLS["chunks among them"], 32, 32, 512, F16, seed=3) for _ in range(2))
    assert np.array_equal(a, b)
