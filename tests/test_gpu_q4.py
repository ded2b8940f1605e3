"""Products of few rows with 4-bit weights (ge_op_gemv_q4, ge_op_gemv_q4_geglu) against float64.

Tolerance. Weights and inputs are exact and products of them exact in fp32 sums; a group's 32 products, its
scale and the sum over the groups each round at 2^-24 of the running magnitude: at most (32 + 2 + K / 32) steps of
2^-24 of sum_k |x| (|d| (q + 8) + |m|), then half a step of y's type. With bf16 x the products are of 16 + q, which
the group's sum then starts from -24 sum_k x or has taken off m: magnitudes up to |d| (q + 40) + |m|. The GeGLU form adds the gate's slope (at most
1.13) and gelu_tanh's own error, a few fp32 steps of its argument's exponent (8 covers exp2 and the reciprocal)."""
import math

import numpy as np
import pytest

import gemma_embed as ge

pytestmark = pytest.mark.gpu
F32, F16, BF16 = ge.GE_TYPE_F32, ge.GE_TYPE_F16, ge.GE_TYPE_BF16
STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TYPES = [ge.GE_TYPE_Q4_0, ge.GE_TYPE_Q4_1]


def to_bits(x, kind):
    f = np.asarray(x, np.float32)
    if kind == F16:
        return f.astype(np.float16).view(np.uint16)
    b = f.view(np.uint32)
    return np.where(np.isnan(f), 0x7fc0, (b + 0x7fff + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def to_float(b, kind):
    if kind == F32:
        return b.astype(np.float64)
    if kind == F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def matrix(rng, kind, rows, cols):
    """(GGUF blocks, float64 weights, float64 |d| (q + 8) + |m|, float64 |d|)."""
    n = rows * cols // 32
    q = rng.integers(0, 16, (n, 32))
    d = (rng.standard_normal(n) * 0.02).astype(np.float16)
    blocks = np.zeros((n, 20 if kind == ge.GE_TYPE_Q4_1 else 18), np.uint8)
    blocks[:, :2] = d.view(np.uint8).reshape(-1, 2)
    blocks[:, -16:] = q[:, :16] | q[:, 16:] << 4
    d = d.astype(np.float64)[:, None]
    if kind == ge.GE_TYPE_Q4_1:
        m = (rng.standard_normal(n) * 0.1).astype(np.float16)
        blocks[:, 2:4] = m.view(np.uint8).reshape(-1, 2)
        m = m.astype(np.float64)[:, None]
        w, size = d * q + m, np.abs(d) * (q + 8) + np.abs(m)
    else:
        w, size = d * (q - 8), np.abs(d) * (q + 8)
    return blocks, w.reshape(rows, cols), size.reshape(rows, cols), np.repeat(np.abs(d), 32, 1).reshape(rows, cols)


def gelu(x):
    return 0.5 * x * (1 + np.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


def product(ctx, kind, m, rows, cols, x_kind, y_kind, geglu=False, seed=0, edit=None):
    rng = np.random.default_rng(seed)
    mats = [matrix(rng, kind, rows, cols) for _ in range(2 if geglu else 1)]
    x = to_bits(rng.standard_normal((m, cols)), x_kind)
    if edit:
        edit(x)
    dtype = np.float32 if y_kind == F32 else np.uint16
    before = rng.integers(0, 100, m * rows + 64).astype(dtype)  # 64 elements past the end stay
    handles = [ctx.q4_create(b, kind, rows, cols) for b, *_ in mats]
    px, py = ctx.alloc(max(x.nbytes, 16)), ctx.alloc(before.nbytes)
    ctx.upload(px, x)
    ctx.upload(py, before)
    (ctx.gemv_q4_geglu if geglu else ctx.gemv_q4)(*handles, px, x_kind, m, py, y_kind)
    raw = ctx.download(py, before.shape, dtype)
    for p in (px, py):
        ctx.free(p)
    for h in handles:
        ctx.q4_destroy(h)
    assert np.array_equal(raw[m * rows:], before[m * rows:])
    f = to_float(x, x_kind)
    y, got = [f @ w.T for _, w, *_ in mats], to_float(raw[:m * rows], y_kind).reshape(m, rows)
    err = [(34 + cols / 32) * 2.0 ** -24 * (np.abs(f) @ (s + 32 * d * (x_kind == BF16)).T) for _, _, s, d in mats]
    if geglu:
        g = gelu(y[0])
        want = g * y[1]
        bound = (1.13 * err[0] + 8 * 2.0 ** -24 * (np.abs(g) + np.abs(y[0]))) * (np.abs(y[1]) + err[1]) + np.abs(g) * err[1]
    else:
        want, bound = y[0], err[0]
    return got, want, bound + STEP[y_kind] * (np.abs(want) + bound) + 2.0 ** -25


def check(*a, **kw):
    got, want, bound = product(*a, **kw)
    over = np.abs(got - want) - bound
    assert over.size == 0 or over.max() <= 0, f"{over.max()} past the bound"


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("x_kind", [F16, BF16])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 150])
@pytest.mark.parametrize("rows,cols", [(1, 32), (17, 64), (40, 160), (129, 1152), (64, 2048)])
def test_shapes(ctx, kind, x_kind, m, rows, cols):
    check(ctx, kind, m, rows, cols, x_kind, F32, seed=m)
    check(ctx, kind, m, rows, cols, x_kind, x_kind, geglu=True, seed=m)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("x_kind", [F16, BF16])
@pytest.mark.parametrize("y_kind", [F32, F16, BF16])
@pytest.mark.parametrize("geglu", [False, True])
def test_types(ctx, kind, x_kind, y_kind, geglu):
    check(ctx, kind, 3, 1001, 768, x_kind, y_kind, geglu=geglu, seed=1)
    check(ctx, kind, 20, 512, 8192, x_kind, y_kind, geglu=geglu, seed=2)


def test_no_rows(ctx):
    check(ctx, ge.GE_TYPE_Q4_0, 0, 64, 64, F16, F32)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("x_kind", [F16, BF16])
def test_not_a_number_stays_in_its_row(ctx, kind, x_kind):
    def edit(x):
        x[3, 5] = 0x7fff

    got, want, bound = product(ctx, kind, 20, 50, 96, x_kind, F32, seed=3, edit=edit)
    assert np.isnan(got[3]).all()
    others = np.arange(20) != 3
    assert (np.abs(got - want) <= bound)[others].all()


@pytest.mark.parametrize("x_kind", [F16, BF16])
def test_largest_inputs(ctx, x_kind):
    """fp16's and bf16's large values: products and sums are fp32."""
    def edit(x):
        x[:] = 0x7bff if x_kind == F16 else 0x7000

    got, want, bound = product(ctx, ge.GE_TYPE_Q4_1, 2, 33, 256, x_kind, F32, seed=4, edit=edit)
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all()


def test_a_rows_bits_do_not_depend_on_its_neighbours(ctx):
    many = product(ctx, ge.GE_TYPE_Q4_0, 64, 96, 1152, F16, F32, seed=5)[0]

    def last(n):
        rng = np.random.default_rng(5)
        blocks, *_ = matrix(rng, ge.GE_TYPE_Q4_0, 96, 1152)
        x = to_bits(rng.standard_normal((64, 1152)), F16)[:n]
        h, px, py = ctx.q4_create(blocks, ge.GE_TYPE_Q4_0, 96, 1152), ctx.alloc(x.nbytes), ctx.alloc(n * 96 * 4)
        ctx.upload(px, x)
        ctx.gemv_q4(h, px, F16, n, py, F32)
        y = ctx.download(py, (n, 96), np.float32)
        ctx.free(px), ctx.free(py), ctx.q4_destroy(h)
        return y

    for n in (1, 16, 20, 63):
        assert np.array_equal(last(n), many[:n])
