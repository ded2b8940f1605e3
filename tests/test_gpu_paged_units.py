"""Rows of heads at any address (ge_op_rotate_heads, ge_op_paged_append) where a wave's lanes leave only some units: head
dims past 256, which move in units of 8, 4 and 1 elements. Against float64; the tolerances of test_gpu_rotary.py."""
import numpy as np
import pytest

import gemma_embed as ge
from test_gpu_causal import BF16, F16, Buffers
from test_gpu_rotary import F32, check, loaded, rotate, stored, turned

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.mark.parametrize("in_type,type", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("hd,dims", [(258, 258), (264, 264), (264, 16), (320, 320), (512, 512), (512, 128), (512, 0)])
@pytest.mark.parametrize("offset", [1, 2, 4])
def test_long_heads_at_any_address(ctx, hd, dims, offset, in_type, type):
    rotate(ctx, 9, 3, 1, hd, in_type, type, dims=dims, normed_heads=3, offset=offset, seed=hd + offset)
    rotate(ctx, 1, 3, 1, hd, in_type, type, dims=dims, layout=1 if dims else 0, offset=offset, seed=hd)


@pytest.mark.parametrize("in_type,type", [(F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("hd,dims", [(64, 64), (264, 132), (512, 512)])
@pytest.mark.parametrize("moved", [1, 2, 4])
def test_an_append_at_any_address(ctx, hd, dims, moved, in_type, type):
    """Inputs, q_out and the pools `moved` elements behind an allocation's start; what lies around the rows stays."""
    heads, kv, page, old, n = 3, 2, 16, 20, 9
    rng = np.random.default_rng(hd + moved)
    counts, order = (heads, kv, kv), [2, 0]
    x = [stored(rng.standard_normal((n, c * hd)), in_type) for c in counts]
    pool = rng.integers(0, 1 << 15, 3 * kv * page * hd + 2 * moved).astype(np.uint16)
    before = rng.integers(0, 1 << 15, n * heads * hd + 2 * moved).astype(np.uint16)
    table, rotary = ctx.page_table_create(1, 2, page, 3), ctx.rotary_create(dims, 1e4)
    ctx.page_table_set(table, [(0, i, p) for i, p in enumerate(order)])
    with Buffers(ctx) as b:
        p = [b.put(np.concatenate([np.zeros(moved, a.dtype), a.ravel()])) + moved * a.itemsize for a in x]
        out, pools = b.put(before), [b.put(pool) for _ in range(2)]
        ctx.paged_append(ge.heads_shape(in_type, type, heads, kv, hd, n), rotary, *p, None, None, None, table, [(0, n, 0, old + n)],
                         out + 2 * moved, pools[0] + 2 * moved, pools[1] + 2 * moved)
        got, cached = ctx.download(out, before.shape, np.uint16), [ctx.download(a, pool.shape, np.uint16) for a in pools]
    ctx.rotary_destroy(rotary)
    ctx.page_table_destroy(table)
    at = np.arange(old, old + n)
    y = [loaded(a, in_type).reshape(n, c, hd) for a, c in zip(x, counts)]
    want, length = turned(y[0], at, dims)
    check(got[moved:-moved].reshape(n, heads, hd), want, length, type, "q")
    assert np.array_equal(got[:moved], before[:moved]) and np.array_equal(got[-moved:], before[-moved:])
    written = np.zeros((3, kv, page, hd), bool)
    for j in at:
        written[order[j // page], :, j % page] = True
    for a, z, turn, name in ((cached[0], y[1], dims, "k"), (cached[1], y[2], 0, "v")):
        want, length = turned(z, at, turn)
        pages = a[moved:-moved].reshape(3, kv, page, hd)
        check(np.stack([pages[order[j // page], :, j % page] for j in at]), want, length, type, name)
        assert np.array_equal(pages[~written], pool[moved:-moved].reshape(3, kv, page, hd)[~written])
        assert np.array_equal(a[:moved], pool[:moved]) and np.array_equal(a[-moved:], pool[-moved:])
