"""The 4-bit products over what x may hold: infinities, NaN, bf16's largest values and fp16's subnormals, at sizes
that take different launch forms. Tolerances are those of test_gpu_q4.py (`product` there): fp32 sums in steps of
2^-24 of the products' magnitudes, then half a step of y's type. Infinities and NaN are those of sum_k x_k w_k
in float64, 0 times infinity among them."""
import numpy as np
import pytest

import gemma_embed as ge
from test_gpu_q4 import BF16, F16, F32, TYPES, gelu, matrix, product, to_bits, to_float

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


BITS = {F16: dict(inf=0x7c00, ninf=0xfc00, nan=0x7e00), BF16: dict(inf=0x7f80, ninf=0xff80, nan=0x7fc0)}
SIZES = [(3, 1001, 160), (7, 70, 96), (20, 1001, 160), (12, 16403, 32), (64, 8195, 32), (20, 4101, 64)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("x_kind", [F16, BF16])
@pytest.mark.parametrize("what", ["inf", "ninf", "nan"])
@pytest.mark.parametrize("m,rows,cols", SIZES)
def test_not_finite(ctx, kind, x_kind, what, m, rows, cols):
    def edit(x):
        x[1, 5], x[m - 1, cols - 1] = BITS[x_kind][what], BITS[x_kind][what]
        x[m - 1, 0] = BITS[x_kind]["inf"]

    with np.errstate(all="ignore"):
        got, want, bound = product(ctx, kind, m, rows, cols, x_kind, F32, seed=3, edit=edit)
    assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN in other places"
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)]), "infinities"
    finite = np.isfinite(want)
    assert (np.abs(got - want)[finite] <= bound[finite]).all()
    assert finite[[i for i in range(m) if i not in (1, m - 1)]].all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("x_kind", [F16, BF16])
def test_geglu_of_infinities(ctx, kind, x_kind):
    """gelu(inf) = inf and gelu(-inf) = NaN (-inf times 0), each times up's own sum."""
    def edit(x):
        x[1, 5] = BITS[x_kind]["inf"]

    for m, rows, cols in ((3, 1001, 160), (20, 1001, 160), (16, 8211, 96)):
        rng = np.random.default_rng(3)
        mats = [matrix(rng, kind, rows, cols) for _ in range(2)]
        x = to_bits(rng.standard_normal((m, cols)), x_kind)
        edit(x)
        got, _, _ = product(ctx, kind, m, rows, cols, x_kind, F32, geglu=True, seed=3, edit=edit)
        with np.errstate(all="ignore"):
            y = [to_float(x, x_kind)[1] @ w.T for _, w, *_ in mats]
            want = gelu(y[0]) * y[1]
        assert np.array_equal(got[1], want, equal_nan=True) and np.isfinite(np.delete(got, 1, 0)).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,rows,cols", SIZES)
def test_bf16s_largest_values(ctx, kind, m, rows, cols):
    """x near bf16's largest, whose integers' products pass fp32's range where y does not."""
    def edit(x):
        x[0, :] = 0x7eff  # 2^127
        x[0, 1::2] = 0xfeff  # the sums cancel in part
        x[2, 3] = 0x7e7f

    got, want, bound = product(ctx, kind, m, rows, cols, BF16, F32, seed=4, edit=edit)
    fits = np.abs(want) < 2.0 ** 127.9
    assert fits[1:].all() and fits[0].mean() > 0.5
    over = (np.abs(got - want) - bound)[fits]
    assert np.isfinite(got[fits]).all() and over.max() <= 0, over.max()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("m,rows,cols", SIZES)
@pytest.mark.parametrize("top", [0x400, 0x40, 0x10])
def test_fp16_subnormals(ctx, kind, m, rows, cols, top):
    """x of subnormals alone: their products keep fp32's precision. y's absolute term is left out of the bound."""
    def edit(x):
        x[:] = np.random.default_rng(5).integers(1, top, x.shape) | np.random.default_rng(6).integers(0, 2, x.shape) << 15

    got, want, bound = product(ctx, kind, m, rows, cols, F16, F32, seed=5, edit=edit)
    over = np.abs(got - want) - (bound - 2.0 ** -25)
    assert over.max() <= 0, (over.max(), (np.abs(got - want) / (bound - 2.0 ** -25)).max())
