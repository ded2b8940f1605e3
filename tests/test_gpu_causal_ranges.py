"""The causal models' attention at the ends of the types' ranges, with the results that follow from the definition.

A row's result is a mean of the values it sees: its weights and their sum are those that the product with V takes,
so where all values are one number the result is that number: the fp32 sums of n weights are off by n 2^-24 at
most, under half a step of either type for n up to 2^12 in fp16 (2^15 in bf16)."""
import numpy as np
import pytest

import gemma_embed as ge
from test_gpu_causal import BF16, F16, LAYOUTS, Buffers, attend, to_bits, to_float

pytestmark = pytest.mark.gpu
# The largest, two ordinary and the smallest normal value; and in bf16 small ones of which the weights' multiples are normal.
CONSTANTS = [(F16, 0x7bff), (F16, 0xfbff), (F16, 0x3c01), (F16, 0x0400), (F16, 0x0003),
             (BF16, 0x7f7f), (BF16, 0xff7f), (BF16, 0x3f81), (BF16, 0x1a01)]


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.mark.parametrize("kind,value", CONSTANTS)
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("scale", [0.1, 1.0])
def test_equal_values_come_out_as_they_are(ctx, heads, kv_heads, hd, kind, value, scale):
    rng = np.random.default_rng(value)
    # a prompt, a chunk, single tokens of one and of several parts
    seqs = [(0, 150, 0, 150), (150, 20, 150, 700), (170, 1, 0, 2000), (171, 1, 10, 33), (172, 1, 5, 1)]
    q, k = (to_bits(rng.standard_normal((n, w * hd)), kind) for n, w in ((173, heads), (2000, kv_heads)))
    v = np.full((2000, kv_heads * hd), value, np.uint16)
    shape = ge.attention_shape(kind, heads, kv_heads, hd, 173, 2000, scale=scale)
    with Buffers(ctx) as b:
        out = b.put(np.zeros((173, heads * hd), np.uint16))
        ctx.attention_causal(shape, b.put(q), b.put(k), b.put(v), seqs, out)
        got = ctx.download(out, (173, heads * hd), np.uint16)
    wrong = np.unique(got[got != value])
    assert not wrong.size, f"{(got != value).mean():.3%} of the results, such as {[hex(x) for x in wrong[:4]]}"


@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
def test_bf16_largest_values_under_rising_scores(ctx, heads, kv_heads, hd):
    """Every key but the first scores 7.9 above it (in log2): the running maximum stays at the first one."""
    def edit(t):
        t["q"][:], t["k"][:], t["v"][:] = 0, 0, 0x7f7f
        t["q"][:, ::hd] = to_bits(np.ones(1), BF16)
        t["k"][1:, ::hd] = to_bits(np.full(1, 7.9 * np.log(2)), BF16)

    got, _ = attend(ctx, [(0, 300, 0, 300), (300, 1, 0, 3000)], heads, kv_heads, hd, BF16, scale=1.0, edit=edit)
    assert (got[:301] == 0x7f7f).all()
