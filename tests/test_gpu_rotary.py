"""Norms and rotary positions of heads (ge_op_rotate_heads) against float64.

Tolerance. With r the length of an element's pair (after the norm, times the magnitude) and all steps in fp32: the norm
sums 512 squares in chains of at most 16 and a tree of 6 (22 roundings, half of them through the root), then
five more roundings: 16 x 2^-24. The angle, reduced in fp64, is rounded to fp32 within half a turn (2^-25 turns, 2^-22.3 of
a radian), its sine and cosine are good to 2^-23, and the products and sums add 4 x 2^-24. Together under 2^-19 r; then one
rounding to the result's type, u relative or fp16's 2^-25."""
import numpy as np
import pytest

import gemma_embed as ge
from test_gpu_causal import BF16, F16, STEP, Buffers, to_bits, to_float

pytestmark = pytest.mark.gpu
F32 = ge.GE_TYPE_F32
EPS = 1e-6


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


def stored(x, kind):
    return x.astype(np.float32) if kind == F32 else to_bits(x, kind)


def loaded(x, kind):
    return x.astype(np.float64) if kind == F32 else to_float(x, kind)


def frequencies(dims, base=1e4, layout=0, scaling=0, factor=1.0, low_turns=1.0, high_turns=4.0, trained=0, magnitude=1.0):
    f = float(np.float32(base)) ** (-2.0 * np.arange(dims // 2) / dims)
    if scaling == ge.GE_ROTARY_LINEAR:
        f = f / factor
    elif scaling == ge.GE_ROTARY_BY_TURNS:
        w = np.clip((trained * f / (2 * np.pi) - low_turns) / (high_turns - low_turns), 0, 1)
        f = f * (w + (1 - w) / factor)
    return f


def turned(x, positions, dims, layout=0, magnitude=1.0, **spec):
    """(rows [n][heads][hd] turned, the length of each element's pair times the magnitude) in float64."""
    y, r = x.copy(), np.abs(x)
    if dims:
        a = np.asarray(positions, np.float64)[:, None] * frequencies(dims, layout=layout, **spec)
        c, s = np.cos(a)[:, None], np.sin(a)[:, None]
        i, j = (np.arange(dims // 2), dims // 2 + np.arange(dims // 2)) if layout == 0 else (np.arange(0, dims, 2), np.arange(1, dims, 2))
        m = float(np.float32(magnitude))
        with np.errstate(all="ignore"):
            y[..., i], y[..., j] = (x[..., i] * c - x[..., j] * s) * m, (x[..., i] * s + x[..., j] * c) * m
            r[..., i] = r[..., j] = np.hypot(x[..., i], x[..., j]) * abs(m)
    return y, r


def normed(x, w, eps=EPS):
    with np.errstate(all="ignore"):
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps)))
    return y if w is None else y * w


def check(got, want, length, kind, what):
    """Results (bits) within the tolerance; infinities and NaN where they should be."""
    y = to_float(got, kind)
    top = 65504.0 if kind == F16 else 3.3895313892515355e38
    with np.errstate(all="ignore"):
        bound = STEP[kind] * np.abs(want) + 2.0 ** -19 * length * (1 + STEP[kind]) + (2.0 ** -25 if kind == F16 else 2.0 ** -134)
        over = np.abs(want) > top * (1 + STEP[kind])  # rounds to infinity
        assert np.array_equal(np.isnan(y), np.isnan(want)), f"{what}: NaN in other places"
        fine = np.isfinite(want) & (np.abs(want) < top)
        assert np.array_equal(y[over], np.sign(want[over]) * np.inf), f"{what}: infinities"
        err = np.abs(y[fine] - want[fine]) - bound[fine]
    assert err.size == 0 or err.max() <= 0, f"{what}: {err.max()} past {bound[fine].max()}"


def rotate(ctx, rows, heads, kv_heads, hd, in_type=None, type=F16, dims=0, normed_heads=0, weights=True, pads=(0, 0, 0, 0), positions=None,
           in_place=False, edit=None, seed=0, eps=EPS, offset=0, **spec):
    rng = np.random.default_rng(seed)
    in_type = type if in_type is None else in_type
    counts = (heads, kv_heads, heads, kv_heads)
    strides = [n * hd + p for n, p in zip(counts, pads)]
    x = [stored(rng.standard_normal((rows, s)), in_type) for s in strides[:2]]
    if edit:
        edit(x)
    w = [1 + 0.1 * rng.standard_normal(hd).astype(np.float32) for _ in range(2)] if weights else [None, None]
    positions = rng.integers(0, 5000, rows) if positions is None else np.asarray(positions)
    before = [rng.integers(0, 1 << 15, (rows, s)).astype(np.uint16) for s in strides[2:]]
    handle = ctx.rotary_create(dims, spec.get("base", 1e4), **{k: v for k, v in spec.items() if k != "base"}) if dims else None
    shape = ge.heads_shape(in_type, type, heads, kv_heads, hd, rows, normed=normed_heads, eps=eps, q_stride=strides[0], k_stride=strides[1],
                           q_out_stride=strides[2], k_out_stride=strides[3])
    with Buffers(ctx) as b:
        def put(a):
            if not offset or a is None:
                return b.put(a) if a is not None and a.size else None
            p = b.put(np.concatenate([np.zeros(offset, a.dtype), a.ravel()]))
            return p + offset * a.itemsize

        p, pw, pos = [put(a) for a in x], [put(a) for a in w], b.put(positions.astype(np.int32)) if dims else None
        out = p if in_place else [put(a) for a in before]
        ctx.rotate_heads(shape, handle, p[0], p[1], pw[0], pw[1], pos, out[0], out[1])
        got = [ctx.download(o, a.shape, np.uint16) if o else a for o, a in zip(out, before)]
    if handle:
        ctx.rotary_destroy(handle)
    for i, name in enumerate("qk"):
        n = counts[i]
        y = loaded(x[i], in_type)[:, :n * hd].reshape(rows, n, hd)
        if normed_heads & (1 << i):
            y = normed(y, None if w[i] is None else w[i].astype(np.float64), eps)
        want, length = turned(y, positions, dims, **spec)
        check(got[i][:, :n * hd].reshape(rows, n, hd), want, length, type, name)
        rest = (x if in_place else before)[i][:, n * hd:]
        assert np.array_equal(got[i][:, n * hd:], rest), f"{name}: elements between the rows changed"
    return got


@pytest.mark.parametrize("in_type,type", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("heads,kv_heads,hd,dims", [(3, 1, 256, 256), (32, 8, 128, 128), (5, 1, 80, 80), (2, 2, 64, 32), (4, 1, 512, 512), (6, 2, 96, 48),
                                                   (2, 1, 16, 16), (1, 1, 32, 16), (7, 3, 34, 34), (2, 1, 72, 24), (1, 2, 512, 130), (3, 1, 128, 2), (1, 1, 2, 2)])
def test_layouts(ctx, heads, kv_heads, hd, dims, layout, in_type, type):
    rotate(ctx, 7, heads, kv_heads, hd, in_type, type, dims, normed_heads=3, layout=layout, seed=hd + dims)
    rotate(ctx, 1, heads, kv_heads, hd, in_type, type, dims, layout=layout, seed=hd)


@pytest.mark.parametrize("in_type,type", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("hd,dims,pad", [(72, 72, 0), (8, 8, 0), (40, 24, 0), (264, 264, 0), (504, 8, 0), (512, 512, 4), (64, 64, 4), (68, 68, 0), (4, 4, 0),
                                         (12, 12, 0), (128, 36, 0), (256, 20, 0), (20, 0, 0), (256, 256, 2), (512, 36, 0), (36, 36, 1)])
def test_units_of_four_and_two(ctx, hd, dims, pad, layout, in_type, type):
    """Heads, parts and strides that come in fewer than 8 elements, some of more units than a wave has lanes."""
    rotate(ctx, 9, 5, 2, hd, in_type, type, dims, normed_heads=3, layout=layout, pads=(pad,) * 4, seed=hd + dims)
    rotate(ctx, 1500, 3, 1, hd, in_type, type, dims, layout=layout, pads=(pad,) * 4, seed=hd)


@pytest.mark.parametrize("normed_heads", [0, 1, 2, 3])
@pytest.mark.parametrize("weights", [True, False])
@pytest.mark.parametrize("hd,dims", [(128, 0), (128, 64), (40, 40), (40, 0)])
def test_norms(ctx, hd, dims, normed_heads, weights):
    rotate(ctx, 19, 5, 2, hd, F32, BF16, dims, normed_heads, weights, seed=normed_heads)
    rotate(ctx, 19, 5, 2, hd, F16, F16, dims, normed_heads, weights, seed=normed_heads)


@pytest.mark.parametrize("heads,kv_heads", [(5, 0), (0, 3), (0, 1), (70, 1), (33, 33)])
@pytest.mark.parametrize("hd", [64, 66])
def test_one_kind_and_many_heads(ctx, heads, kv_heads, hd):
    rotate(ctx, 5, heads, kv_heads, hd, dims=64, normed_heads=3)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 1001, 8192, 8193, 20001])
@pytest.mark.parametrize("hd", [64, 50])
def test_rows(ctx, rows, hd):
    rotate(ctx, rows, 2, 1, hd, F32, BF16, dims=hd, normed_heads=3, seed=rows)


@pytest.mark.parametrize("spec", [dict(scaling=1, factor=4.0), dict(scaling=2, factor=8.0, trained=8192), dict(scaling=2, factor=8.0, trained=8192, base=5e5),
                                  dict(magnitude=1.2), dict(magnitude=0.3, layout=1), dict(base=1e6), dict(base=0.5),
                                  dict(scaling=2, factor=2.0, trained=100, low_turns=-3.0, high_turns=0.5)])
def test_scalings(ctx, spec):
    for hd in (128, 36):
        rotate(ctx, 40, 2, 1, hd, F32, F16, dims=hd, positions=np.arange(40) * 2003, **spec)


@pytest.mark.parametrize("layout", [0, 1])
def test_far_positions(ctx, layout):
    """Angles of positions up to 2^31 keep fp32's accuracy; negative ones turn back."""
    at = [0, 1, 2, -1, -7, 65535, 1 << 20, (1 << 24) + 1, (1 << 30) + 12345, (1 << 31) - 1, -(1 << 31), 99999999]
    for hd in (128, 22):
        rotate(ctx, len(at), 3, 1, hd, F32, F16, dims=hd, positions=at, layout=layout)
        rotate(ctx, len(at), 3, 1, hd, F32, F16, dims=hd, positions=at, layout=layout, scaling=1, factor=32.0, normed_heads=3)


@pytest.mark.parametrize("pads", [(8, 16, 24, 8), (128, 0, 0, 64), (1, 3, 5, 7), (0, 2, 0, 0), (4, 4, 8, 8)])
@pytest.mark.parametrize("in_type", [F32, F16])
def test_strides(ctx, pads, in_type):
    rotate(ctx, 9, 3, 1, 64, in_type, F16, dims=64, normed_heads=3, pads=pads)


@pytest.mark.parametrize("offset", [1, 2, 3, 4])
def test_addresses(ctx, offset):
    """Buffers at any element."""
    rotate(ctx, 9, 3, 1, 64, F32, BF16, dims=64, normed_heads=3, offset=offset)
    rotate(ctx, 9, 3, 1, 64, F16, F16, dims=32, normed_heads=3, offset=offset)


@pytest.mark.parametrize("hd,dims", [(128, 128), (64, 48), (34, 20)])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("type", [F16, BF16])
def test_in_place(ctx, hd, dims, layout, type):
    rotate(ctx, 1030, 4, 2, hd, type, type, dims=dims, normed_heads=3, layout=layout, in_place=True, pads=(8, 16, 8, 16))


def test_one_projections_output_in_place(ctx):
    """q and k as views of one buffer, turned where they are; v beside them stays."""
    heads, kv, hd, n = 4, 2, 128, 33
    width = (heads + 2 * kv) * hd
    x = to_bits(np.random.default_rng(4).standard_normal((n, width)), F16)
    h = ctx.rotary_create(hd, 1e4)
    shape = ge.heads_shape(F16, F16, heads, kv, hd, n, q_stride=width, k_stride=width, q_out_stride=width, k_out_stride=width)
    with Buffers(ctx) as b:
        p, pos = b.put(x), b.put(np.arange(n, dtype=np.int32))
        ctx.rotate_heads(shape, h, p, p + heads * hd * 2, None, None, pos, p, p + heads * hd * 2)
        got = ctx.download(p, x.shape, np.uint16)
    ctx.rotary_destroy(h)
    want, length = turned(to_float(x, F16).reshape(n, -1, hd)[:, :heads + kv], np.arange(n), hd)
    check(got[:, :(heads + kv) * hd].reshape(n, -1, hd), want, length, F16, "q and k")
    assert np.array_equal(got[:, (heads + kv) * hd:], x[:, (heads + kv) * hd:])


@pytest.mark.parametrize("hd", [128, 40])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_norms_of_the_largest_and_smallest(ctx, hd, eps):
    """Rows whose squares leave fp32's range, or fall below it, are normed all the same."""
    def edit(x):
        for t, row in ((x[0], 0), (x[1], 1)):
            t[row] *= 1e30
            t[row + 2] *= 1e37
            t[row + 4] *= 1e-25
            t[row + 6] *= 1e-12
            t[row + 8, 1:] = 0
    rotate(ctx, 12, 3, 2, hd, F32, BF16, dims=hd // 4 * 2, normed_heads=3, edit=edit, eps=eps)


@pytest.mark.parametrize("hd", [128, 40])
@pytest.mark.parametrize("layout", [0, 1])
def test_infinities_and_nan(ctx, hd, layout):
    """They stay in their pair, or with a norm in their head; what does not turn is copied."""
    def edit(x):
        for t in x:
            t[0, 3], t[1, hd - 1], t[2, hd + 1] = np.inf, -np.inf, np.nan
    for normed_heads in (0, 3):
        rotate(ctx, 5, 3, 2, hd, F32, F16, dims=16, normed_heads=normed_heads, edit=edit, layout=layout, positions=[5, 6, 7, 8, 9])


@pytest.mark.parametrize("type", [F16, BF16])
def test_the_largest_values(ctx, type):
    """A turn brings a value past the type's largest to infinity, and none before that."""
    top = 65504.0 if type == F16 else 3.3895313892515355e38

    def edit(x):
        for t in x:
            t[:] = to_bits(np.where(np.arange(t.size).reshape(t.shape) % 3 == 0, -top, top), type)
    for magnitude in (1.0, 0.5, 1.2):
        rotate(ctx, 50, 2, 1, 64, type=type, dims=64, edit=edit, magnitude=magnitude, positions=np.arange(50) * 37)


def test_nothing_to_turn_is_a_copy(ctx):
    got = rotate(ctx, 33, 3, 2, 64, BF16, BF16)
    assert len(got) == 2
    rotate(ctx, 33, 3, 2, 64, F32, F16)


def test_the_same_bits_every_time(ctx):
    a, b = (rotate(ctx, 300, 8, 2, 128, F32, BF16, dims=128, normed_heads=3, seed=3) for _ in range(2))
    assert all(np.array_equal(x, y) for x, y in zip(a, b))
