"""Attention over a shared prefix where the texts' rows stack up over it (tests/causal_stacked.py) against float64.
Tolerances as in test_gpu_causal.py."""
import numpy as np
import pytest

import gemma_embed as ge
from causal_stacked import STACKED
from test_gpu_causal import BF16, BITS, F16, Buffers, attend, to_bits, to_float

pytestmark = pytest.mark.gpu


def some(*names):
    calls = [c for c in STACKED if not names or c[0] in names]
    return calls, False, [f"{c[0]}-{c[1]}-{c[2]}-{c[3]}" for c in calls]


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("name,heads,kv_heads,hd,prefix,seqs", *some())
def test_stacked(ctx, name, heads, kv_heads, hd, prefix, seqs, kind):
    attend(ctx, seqs, heads, kv_heads, hd, kind, prefix=prefix, seed=40)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("name,heads,kv_heads,hd,prefix,seqs", *some("tokens", "mixed"))
def test_strides_and_a_negative_scale(ctx, name, heads, kv_heads, hd, prefix, seqs, kind):
    attend(ctx, seqs, heads, kv_heads, hd, kind, prefix=prefix, seed=41, pads=(8, 64, 200, 16), scale=-0.2)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("name,heads,kv_heads,hd,prefix,seqs", *some("tokens", "mixed", "apart"))
def test_infinities_in_the_prefix_and_beside_own_keys(ctx, name, heads, kv_heads, hd, prefix, seqs, kind):
    """A value of the prefix reaches every row that sees it, one of a text's own rows that text's later rows."""
    last = max(s[2] + s[3] for s in seqs)

    def edit(t):
        t["pv"][7, 1], t["pv"][prefix - 1, hd - 1] = BITS[kind]["inf"], BITS[kind]["nan"]
        if last:
            t["v"][last - 1, 0], t["v"][last // 2, 2] = BITS[kind]["ninf"], BITS[kind]["inf"]

    got, _ = attend(ctx, seqs, heads, kv_heads, hd, kind, prefix=prefix, seed=42, edit=edit, scale=0.02)
    first = to_float(got[seqs[1][0]], kind)
    assert first[1] == np.inf and np.isnan(first[hd - 1]) and np.isfinite(first[3:hd - 1]).all()


@pytest.mark.parametrize("kind", [F16, BF16])
def test_large_calls_repeat_bitwise(ctx, kind):
    """Calls that fill the GPU: wide and narrow items, split ones, a window, a stacked prefix."""
    rng = np.random.default_rng(30)
    for heads, kv_heads, hd, window, prefix, seqs in (
            (32, 8, 128, 0, 0, [(i, 1, 700 * i, 300 + 9 * i) for i in range(48)]),
            (16, 16, 64, 0, 0, [(0, 512, 0, 4000), (512, 512, 4000, 3000)]),
            (3, 1, 256, 512, 0, [(700 * i, 700, 700 * i, 700) for i in range(6)]),
            (3, 1, 256, 0, 4000, [(40 * i, 40, 40 * i, 40) for i in range(64)])):
        n, m = seqs[-1][0] + seqs[-1][1], seqs[-1][2] + seqs[-1][3]
        arrays = [to_bits(rng.standard_normal((r, w * hd)), kind) for r, w in ((n, heads), (m, kv_heads), (m, kv_heads), (prefix, kv_heads), (prefix, kv_heads))]
        shape = ge.attention_shape(kind, heads, kv_heads, hd, n, m, scale=hd ** -0.5, window=window)
        with Buffers(ctx) as b:
            q, k, v, pk, pv = (b.put(a) for a in arrays)
            out, results = b.put(np.zeros((n, heads * hd), np.uint16)), []
            for _ in range(4):
                ctx.upload(out, np.full((n, heads * hd), 0x7e7e, np.uint16))
                ctx.attention_prefix(shape, q, pk, pv, prefix, k, v, seqs, out)
                results.append(ctx.download(out, (n, heads * hd), np.uint16))
        assert all(np.array_equal(r, results[0]) for r in results[1:]) and np.isfinite(to_float(results[0], kind)).all()
