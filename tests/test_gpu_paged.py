"""A paged cache (ge_op_paged_append, ge_op_attention_paged) against float64.

Appending: the tolerances of test_gpu_rotary.py. Attention: those of test_gpu_causal.py, and a cap's: its tanh
is off by 2^-21.5 (its exponential by 2^-23 and its argument's rounding, a third of 2^-24 at most after the
slope; the reciprocal 2^-23 twice, the last sum 2^-24), so a score by e_cap = cap 2^-21, which is added to the scores'
own error e."""
import threading

import numpy as np
import pytest

import gemma_embed as ge
from test_gpu_causal import BF16, F16, LAYOUTS, STEP, Buffers, reference, to_bits, to_float
from test_gpu_rotary import EPS, F32, check, loaded, normed, stored, turned

pytestmark = pytest.mark.gpu
NAN = {F16: 0x7e00, BF16: 0x7fc0}
INF = {F16: 0x7c00, BF16: 0x7f80}


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


class Cache:
    """A pool of pages in host memory, NaN wherever no key is, and a table of which pages hold which keys."""

    def __init__(self, ctx, rng, lengths, page, kv_heads, hd, kind, gap=0, values=1.0, freed=()):
        self.ctx, self.page, self.kind, self.kv_heads, self.hd = ctx, page, kind, kv_heads, hd
        counts = [-(-n // page) for n in lengths]
        self.n_pages = sum(counts) + 3
        order = rng.permutation(self.n_pages)
        self.elements = page * kv_heads * hd
        self.stride = self.elements + gap
        self.table = np.full((len(lengths), max(counts + [1])), -1, np.int64)
        self.k, self.v = (np.full((self.n_pages, self.stride), NAN[kind], np.uint16) for _ in range(2))
        at = 0
        for s, n in enumerate(lengths):
            self.table[s, :counts[s]] = order[at:at + counts[s]]
            at += counts[s]
            for j in range(n):
                for pool, mul in ((self.k, 1.0), (self.v, values)):
                    self.row(pool, s, j)[:] = to_bits(rng.standard_normal((kv_heads, hd)) * mul, kind)
        self.handle = ctx.page_table_create(*self.table.shape, page, self.n_pages)
        slots, index = np.nonzero(self.table >= 0)
        ctx.page_table_set(self.handle, np.stack([slots, index, self.table[slots, index]], 1))

    def row(self, pool, slot, key):
        """[kv_heads][hd] of one key, a view."""
        p = self.table[slot, key // self.page]
        return pool[p, :self.elements].reshape(self.kv_heads, self.page, self.hd)[:, key % self.page]

    def rows(self, pool, slot, first, end):
        """Keys [first, end) as float64 [keys][kv_heads][hd]."""
        out = [self.row(pool, slot, j) for j in range(first, end)]
        return to_float(np.stack(out), self.kind) if out else np.zeros((0, self.kv_heads, self.hd))

    def close(self):
        self.ctx.page_table_destroy(self.handle)


def capped_reference(q, k, v, scale, window, cap):
    """test_gpu_causal's reference with capped scores."""
    if not cap:
        return reference(q, k, v, scale, window)
    n, heads, _ = q.shape
    m, group = len(k), heads // k.shape[1]
    ahead = np.arange(m)[None, :] - np.arange(n)[:, None] - (m - n)
    hidden = ahead > 0
    if window:
        hidden |= ahead <= -window
    o, mag = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(heads):
        with np.errstate(all="ignore"):
            s = np.where(hidden, -np.inf, cap * np.tanh(scale * (q[:, h] @ k[:, h // group].T) / cap))
        top = s.max(1, keepdims=True, initial=-np.inf)
        p = np.where(hidden, 0.0, np.exp(s - np.where(top == -np.inf, 0.0, top)))
        p = p / np.where(p.sum(1, keepdims=True) == 0, 1.0, p.sum(1, keepdims=True))
        for i in range(n):  # hidden values do not count
            seen = ~hidden[i]
            o[i, h], mag[i, h] = p[i, seen] @ v[seen, h // group], p[i, seen] @ np.abs(v[seen, h // group])
    return o, mag


def attend(ctx, seqs, heads, kv_heads, hd, kind, page=16, window=0, scale=None, cap=0.0, seed=0, pads=(0, 0), gap=0, spare=3, edit=None,
           values=1.0, slots=None, interleave=False):
    """One call; seqs: (q_start, q_len, kv_len), each with a slot of its own, checked against the reference."""
    rng = np.random.default_rng(seed)
    scale = hd ** -0.5 if scale is None else scale
    cache = Cache(ctx, rng, [m for _, _, m in seqs], page, kv_heads, hd, kind, gap, values)
    q_rows = max([s[0] + s[1] for s in seqs] + [0]) + spare
    strides = [heads * hd + p for p in pads]
    q = to_bits(rng.standard_normal((q_rows, strides[0])), kind)
    if edit:
        edit(q, cache)
    before = rng.integers(0, 1 << 15, (q_rows, strides[1])).astype(np.uint16)
    order = list(range(len(seqs)))
    call = [(s[0], s[1], i, s[2]) for i, s in zip(order, seqs)]
    with Buffers(ctx) as b:
        if interleave:  # K and V by turns in one buffer
            both = b.put(np.stack([cache.k, cache.v], 1))
            pk, pv, page_stride = both, both + cache.stride * 2, 2 * cache.stride
        else:
            pk, pv, page_stride = b.put(cache.k), b.put(cache.v), cache.stride
        shape = ge.paged_shape(kind, heads, kv_heads, hd, q_rows, scale=scale, window=window, cap=cap, q_stride=strides[0],
                               out_stride=strides[1], page_stride=page_stride)
        pq, out = b.put(q), b.put(before)
        ctx.attention_paged(shape, pq, cache.handle, pk, pv, call, out)
        got = ctx.download(out, before.shape, np.uint16)
    cache.close()
    untouched = np.ones(before.shape, bool)
    f = to_float(q, kind)
    for i, (q0, n, m) in enumerate(seqs):
        untouched[q0:q0 + n, :heads * hd] = False
        if n == 0:
            continue
        x = f[q0:q0 + n, :heads * hd].reshape(n, heads, hd)
        ks, vs = cache.rows(cache.k, i, 0, m), cache.rows(cache.v, i, 0, m)
        o, mag = capped_reference(x, ks, vs, scale, window, cap)
        with np.errstate(all="ignore"):
            big = abs(scale) * np.sqrt((x ** 2).sum(-1).max() * (ks ** 2).sum(-1).max()) if m else 0.0
            big = big if np.isfinite(big) else 1.0
            e = 2 * hd * 2.0 ** -24 * big + cap * 2.0 ** -21
            u = STEP[kind]
            bound = (u + 2 * e + m * 2.0 ** -31) * mag + u * np.abs(o) + 1e-7
        y = to_float(got[q0:q0 + n, :heads * hd], kind).reshape(n, heads, hd)
        finite = np.isfinite(o)
        assert np.array_equal(np.isnan(y), np.isnan(o)), f"sequence {i}: NaN in other places"
        assert np.array_equal(y[np.isinf(o)], o[np.isinf(o)]), f"sequence {i}: infinities"
        over = np.abs(y[finite] - o[finite]) - bound[finite]
        assert over.size == 0 or over.max() <= 0, f"sequence {i}: {over.max()} past {bound[finite].max()}"
    assert np.array_equal(got[untouched], before[untouched]), "rows or columns outside the sequences changed"
    return got


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("page", [8, 16, 64, 256])
def test_tokens(ctx, heads, kv_heads, hd, kind, page):
    seqs = [(i, 1, m) for i, m in enumerate([1, 2, 7, 8, 9, 31, 32, 33, 127, 128, 129, 700, 2049])]
    attend(ctx, seqs, heads, kv_heads, hd, kind, page, seed=page)
    attend(ctx, seqs, heads, kv_heads, hd, kind, page, window=100, seed=page)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("page", [8, 32, 128])
@pytest.mark.parametrize("window", [0, 1, 5, 77, 200])
def test_chunks(ctx, heads, kv_heads, hd, kind, page, window):
    seqs = [(0, 5, 800), (6, 40, 41), (50, 130, 500), (180, 0, 10), (180, 1, 1), (190, 70, 70)]
    attend(ctx, seqs, heads, kv_heads, hd, kind, page, window=window, seed=window)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("n", [1, 31, 33, 64, 65, 129, 300])
def test_prompts(ctx, heads, kv_heads, hd, kind, n):
    attend(ctx, [(0, n, n)], heads, kv_heads, hd, kind, seed=n)


@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
def test_queries_before_their_first_key(ctx, heads, kv_heads, hd):
    got = attend(ctx, [(0, 9, 4), (9, 3, 0), (12, 200, 60)], heads, kv_heads, hd, F16)
    assert not got[:5].any() and not got[9:12].any() and not got[12:152].any()
    attend(ctx, [(0, 9, 4), (9, 3, 0), (12, 200, 60)], heads, kv_heads, hd, BF16, window=3, cap=5.0)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("cap,scale", [(50.0, 1.0), (5.0, 1.0), (0.01, 3.0), (256.0, 1.0), (257.0, 1.0), (1024.0, 1.0), (50.0, -0.7), (50.0, 0.0), (1e-30, 1.0)])
def test_caps(ctx, heads, kv_heads, hd, kind, cap, scale):
    attend(ctx, [(0, 70, 200), (70, 1, 333), (71, 9, 9)], heads, kv_heads, hd, kind, cap=cap, scale=scale, seed=7)
    attend(ctx, [(0, 40, 200), (40, 1, 333)], heads, kv_heads, hd, kind, cap=cap, scale=scale, window=33, seed=8)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales(ctx, kind, scale):
    for layout in LAYOUTS:
        attend(ctx, [(0, 70, 70), (70, 1, 200)], *layout, kind, scale=scale, seed=7)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
def test_strides_and_pages_apart(ctx, heads, kv_heads, hd, kind):
    seqs = [(1, 40, 90), (41, 1, 300)]
    attend(ctx, seqs, heads, kv_heads, hd, kind, pads=(8, 64), gap=24)
    attend(ctx, seqs, heads, kv_heads, hd, kind, pads=(200, 16), interleave=True)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("window", [0, 3, 37, 150])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_hidden_infinities_and_nan(ctx, heads, kv_heads, hd, kind, window, cap):
    """Keys before a window, after a row's position and past the end hold NaN and infinities; values that some rows see."""
    def edit(q, cache):
        for s, j, x in ((0, 110, INF), (0, 122, NAN), (1, 199, NAN), (2, 60, INF)):
            cache.row(cache.v, s, j)[0, 1] = x[kind]
        if window:
            for s, n in ((0, 123 - 20), (1, 200), (2, 61 - 3)):
                for j in range(max(0, n - window + (1 if s != 1 else 0))):
                    cache.row(cache.k, s, j)[:] = NAN[kind]
                    cache.row(cache.v, s, j)[:] = INF[kind]

    seqs = [(0, 20, 123), (20, 1, 200), (25, 3, 61)]
    attend(ctx, seqs, heads, kv_heads, hd, kind, window=window, cap=cap, seed=21, edit=edit)


@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("n", [1, 30])
def test_pages_taken_out_before_a_window(ctx, heads, kv_heads, hd, n):
    """What lies before a window's reach may be gone: the page with its first key may begin with others."""
    rng = np.random.default_rng(1)
    m, window, page = 500, 150, 32
    cache = Cache(ctx, rng, [m], page, kv_heads, hd, F16)
    low = m - n - window + 1
    q = to_bits(rng.standard_normal((n, heads * hd)), F16)
    with Buffers(ctx) as b:
        shape = ge.paged_shape(F16, heads, kv_heads, hd, n, scale=0.1, window=window)
        args = (b.put(q), cache.handle, b.put(cache.k), b.put(cache.v), [(0, n, 0, m)])
        out = [b.put(np.zeros_like(q)) for _ in range(2)]
        ctx.attention_paged(shape, *args, out[0])
        ctx.page_table_set(cache.handle, [(0, i, -1) for i in range(low // page)])
        ctx.attention_paged(shape, *args, out[1])
        a, c = (ctx.download(o, q.shape, np.uint16) for o in out)
        assert np.array_equal(a, c) and a.any()
        ctx.page_table_set(cache.handle, [(0, low // page, -1)])
        with pytest.raises(ge.GemmaEmbedError):
            ctx.attention_paged(shape, *args, out[1])
    cache.close()


@pytest.mark.parametrize("hd", [64, 256])
def test_the_largest_values(ctx, hd):
    """A mean of values that are all the type's largest is that."""
    for kind, bits in ((F16, 0x7bff), (BF16, 0x7f7f)):
        def edit(q, cache):
            for pool in (cache.v,):
                for s, n in ((0, 300), (1, 2000)):
                    for j in range(n):
                        cache.row(pool, s, j)[:] = bits
        got = attend(ctx, [(0, 100, 300), (100, 1, 2000)], 2, 1, hd, kind, edit=edit, scale=0.3)
        assert (got[:101, :2 * hd] == bits).all()


def test_a_row_does_not_depend_on_its_neighbours_or_pages(ctx):
    """The same keys in pages of other sizes, and beside other sequences: the same bits."""
    heads, kv, hd, n, m = 4, 1, 128, 40, 300
    rng = np.random.default_rng(9)
    k, v, q = (to_bits(rng.standard_normal(s), BF16) for s in ((m, kv, hd), (m, kv, hd), (n, heads * hd)))
    results = []
    for page in (8, 64, 512):
        cache = Cache(ctx, rng, [m, 50], page, kv, hd, BF16)
        for j in range(m):
            cache.row(cache.k, 0, j)[:], cache.row(cache.v, 0, j)[:] = k[j], v[j]
        with Buffers(ctx) as b:
            shape = ge.paged_shape(BF16, heads, kv, hd, n, scale=0.1)
            out = b.put(np.zeros_like(q))
            ctx.attention_paged(shape, b.put(q), cache.handle, b.put(cache.k), b.put(cache.v), [(0, n, 0, m)], out)
            results.append(ctx.download(out, q.shape, np.uint16))
        cache.close()
    with Buffers(ctx) as b:  # and as attention over rows has them
        shape = ge.attention_shape(BF16, heads, kv, hd, n, m, scale=0.1)
        out = b.put(np.zeros_like(q))
        ctx.attention_causal(shape, b.put(q), b.put(k), b.put(v), [(0, n, 0, m)], out)
        results.append(ctx.download(out, q.shape, np.uint16))
    f = to_float(results[-1], BF16)
    assert all(np.array_equal(r, results[0]) for r in results[1:3])
    assert np.abs(to_float(results[0], BF16) - f).max() <= 2 * STEP[BF16] * np.abs(f).max()


def test_slots_that_share_pages_and_one_slot_twice(ctx):
    heads, kv, hd, page = 2, 1, 64, 16
    rng = np.random.default_rng(2)
    cache = Cache(ctx, rng, [160, 160], page, kv, hd, F16)
    ctx.page_table_set(cache.handle, [(1, i, cache.table[0, i]) for i in range(10)])
    q = to_bits(rng.standard_normal((1, heads * hd)), F16)
    q = np.repeat(q, 4, 0)
    with Buffers(ctx) as b:
        out = b.put(np.zeros_like(q))
        shape = ge.paged_shape(F16, heads, kv, hd, 4, scale=0.1)
        ctx.attention_paged(shape, b.put(q), cache.handle, b.put(cache.k), b.put(cache.v), [(0, 1, 0, 160), (1, 1, 1, 160), (2, 1, 0, 160), (3, 1, 0, 150)], out)
        got = ctx.download(out, q.shape, np.uint16)
    cache.close()
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2]) and not np.array_equal(got[0], got[3])


def test_long_caches(ctx):
    """Many parts to join, and a short sequence beside a long one."""
    attend(ctx, [(0, 1, 9000), (1, 1, 3), (2, 33, 6000)], 4, 1, 64, F16, page=64, seed=11)
    attend(ctx, [(0, 1, 5001), (1, 2, 5000)], 2, 1, 512, BF16, page=16, seed=12)


# ---------------------------------------------------------------------------- appending


def append(ctx, seqs, heads, kv_heads, hd, in_type=None, type=F16, page=16, dims=0, normed_heads=0, fused=False, gap=0, positions=None,
           in_place=False, seed=0, spare=3, **spec):
    """seqs: (q_start, q_len, kv_len), each with a slot of its own."""
    rng = np.random.default_rng(seed)
    in_type = type if in_type is None else in_type
    cache = Cache(ctx, rng, [m for _, _, m in seqs], page, kv_heads, hd, type, gap)
    rows = max([s[0] + s[1] for s in seqs] + [0]) + spare
    counts = [heads, kv_heads, kv_heads]
    x = stored(rng.standard_normal((rows, sum(counts) * hd)), in_type)
    parts = np.split(x, np.cumsum([n * hd for n in counts])[:2], 1)
    w = [1 + 0.1 * rng.standard_normal(hd).astype(np.float32) for _ in range(2)]
    before = rng.integers(0, 1 << 15, (rows, heads * hd)).astype(np.uint16)
    handle = ctx.rotary_create(dims, spec.get("base", 1e4), **{k: v for k, v in spec.items() if k != "base"}) if dims else None
    width = x.shape[1] if fused else 0
    shape = ge.heads_shape(in_type, type, heads, kv_heads, hd, rows, normed=normed_heads, eps=EPS, q_stride=width, k_stride=width,
                           v_stride=width, q_out_stride=width if in_place else 0, page_stride=cache.stride)
    size = x.itemsize
    with Buffers(ctx) as b:
        if fused:
            p = b.put(x)
            q, k, v = p, p + heads * hd * size, p + (heads + kv_heads) * hd * size
        else:
            q, k, v = (b.put(np.ascontiguousarray(a)) if a.size else None for a in parts)
        pk, pv = b.put(cache.k), b.put(cache.v)
        q_out = q if in_place else b.put(before)
        pos = None if positions is None else b.put(np.asarray(positions, np.int32))
        ctx.paged_append(shape, handle, q, k, v, b.put(w[0]), b.put(w[1]), pos, cache.handle, [(s[0], s[1], i, s[2]) for i, s in enumerate(seqs)],
                         q_out, pk, pv)
        got = ctx.download(q_out, (rows, width) if in_place else before.shape, np.uint16)[:, :heads * hd]
        pools = [ctx.download(p, cache.k.shape, np.uint16) for p in (pk, pv)]
    if handle:
        ctx.rotary_destroy(handle)
    kept = x[:, :heads * hd] if in_place else before
    untouched = np.ones(rows, bool)
    written = np.zeros(cache.k.shape, bool)
    for i, (q0, n, m) in enumerate(seqs):
        at = np.arange(m - n, m) if positions is None else np.asarray(positions)[q0:q0 + n]
        untouched[q0:q0 + n] = False
        y = [loaded(a[q0:q0 + n], in_type).reshape(n, c, hd) for a, c in zip(parts, counts)]
        for j, weight in enumerate([w[0], w[1], None]):
            if normed_heads & (1 << j):
                y[j] = normed(y[j], None if weight is None else weight.astype(np.float64))
        want, length = turned(y[0], at, dims, **spec)
        check(got[q0:q0 + n].reshape(n, heads, hd), want, length, type, f"sequence {i}: q")
        for pool, z, name, turn in ((pools[0], y[1], "k", dims), (pools[1], y[2], "v", 0)):
            want, length = turned(z, at, turn, **(spec if turn else {}))
            rows_got = np.stack([cache.row(pool, i, j) for j in range(m - n, m)]) if n else np.zeros((0, kv_heads, hd), np.uint16)
            check(rows_got, want, length, type, f"sequence {i}: {name}")
        for j in range(m - n, m):
            cache.row(written, i, j)[:] = True
    assert np.array_equal(got[untouched], kept[untouched]), "rows of q outside the sequences changed"
    for pool, old, name in ((pools[0], cache.k, "k"), (pools[1], cache.v, "v")):
        assert np.array_equal(pool[~written], old[~written]), f"other rows of {name}'s pages changed"
    cache.close()


SEQS = [(0, 5, 5), (5, 0, 40), (7, 1, 300), (8, 40, 77), (50, 1, 1), (51, 33, 64)]


@pytest.mark.parametrize("in_type,type", [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("heads,kv_heads,hd,dims", [(3, 1, 256, 256), (8, 2, 128, 128), (4, 1, 512, 512), (12, 4, 64, 32), (5, 1, 80, 80), (2, 2, 34, 20),
                                                   (2, 1, 72, 24), (0, 2, 64, 64), (2, 1, 128, 0)])
@pytest.mark.parametrize("page", [8, 16, 128])
def test_appending(ctx, heads, kv_heads, hd, dims, in_type, type, page):
    append(ctx, SEQS, heads, kv_heads, hd, in_type, type, page, dims, normed_heads=7, seed=page)
    append(ctx, SEQS, heads, kv_heads, hd, in_type, type, page, dims, fused=True, layout=1 if dims else 0, seed=page) if dims else None


@pytest.mark.parametrize("in_type,type", [(F32, BF16), (F16, F16)])
@pytest.mark.parametrize("hd,dims", [(72, 72), (40, 40), (40, 20), (128, 36), (64, 20), (12, 12), (8, 8), (4, 4), (264, 132), (512, 36)])
def test_appending_in_units_of_four_and_two(ctx, hd, dims, in_type, type):
    append(ctx, SEQS, 5, 2, hd, in_type, type, 8, dims, normed_heads=7, fused=True, seed=hd)
    append(ctx, SEQS, 5, 2, hd, in_type, type, 32, dims, layout=1, seed=dims)


@pytest.mark.parametrize("normed_heads", range(8))
def test_norms_of_an_append(ctx, normed_heads):
    append(ctx, SEQS, 4, 2, 128, F32, BF16, dims=64, normed_heads=normed_heads, fused=True, seed=normed_heads)


@pytest.mark.parametrize("hd", [64, 36])
def test_positions_other_than_the_cache_row(ctx, hd):
    positions = np.random.default_rng(5).integers(-1000, 1 << 30, 87)
    append(ctx, SEQS, 4, 2, hd, F32, F16, dims=hd, positions=positions, scaling=1, factor=8.0, magnitude=1.1)


@pytest.mark.parametrize("type", [F16, BF16])
def test_queries_turned_in_place(ctx, type):
    append(ctx, SEQS, 4, 2, 64, type, type, dims=64, normed_heads=7, fused=True, in_place=True)


def test_pages_of_a_stride(ctx):
    append(ctx, SEQS, 4, 2, 64, F32, F16, dims=64, gap=40)
    append(ctx, SEQS, 4, 2, 66, F32, F16, dims=64, gap=8)


def test_many_sequences(ctx):
    append(ctx, [(i, 1, 1 + 7 * i % 40) for i in range(300)], 4, 2, 64, F16, F16, dims=64)
    append(ctx, [(3 * i, 2, 2 + i % 9) for i in range(260)], 1, 1, 32, F32, BF16, dims=32, normed_heads=7)


def test_a_refused_append_writes_nothing(ctx):
    rng = np.random.default_rng(3)
    cache = Cache(ctx, rng, [40, 40], 16, 1, 64, F16)
    ctx.page_table_set(cache.handle, [(1, 2, cache.table[0, 2])])
    x = to_bits(rng.standard_normal((4, 64)), F16)
    with Buffers(ctx) as b:
        p, pk, pv, out = b.put(x), b.put(cache.k), b.put(cache.v), b.put(np.zeros_like(x))
        for seqs in ([(0, 1, 0, 40), (1, 1, 1, 39)], [(0, 1, 0, 40), (1, 1, 1, 60)], [(0, 1, 0, 40), (1, 3, 1, 2)]):
            with pytest.raises(ge.GemmaEmbedError) as e:
                ctx.paged_append(ge.heads_shape(F16, F16, 1, 1, 64, 4), None, p, p, p, None, None, None, cache.handle, seqs, out, pk, pv)
            assert e.value.code == ge.GE_ERR_INVALID
        assert np.array_equal(ctx.download(pk, cache.k.shape, np.uint16), cache.k) and not ctx.download(out, x.shape, np.uint16).any()
    cache.close()


# ---------------------------------------------------------------------------- together


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd,window,cap", [(3, 1, 256, 40, 0.0), (8, 2, 128, 0, 0.0), (4, 2, 64, 0, 30.0), (2, 1, 512, 70, 50.0)])
def test_texts_read_in_pieces(ctx, type, heads, kv_heads, hd, window, cap):
    """A server's loop: prompts, chunks and single tokens of several texts by turns, pages given out as they are needed and
    taken back behind the window; every step's attention against float64 over the keys so far, and, without window
    and cap, against attention over the same keys row after row."""
    rng = np.random.default_rng(17)
    page, slots, n_pages = 16, 3, 64
    free, held = list(rng.permutation(n_pages)), {s: {} for s in range(slots)}
    table = ctx.page_table_create(slots, 32, page, n_pages)
    rotary = ctx.rotary_create(hd, 1e4)
    lengths, keys, values = [0] * slots, [[] for _ in range(slots)], [[] for _ in range(slots)]
    scale = hd ** -0.5 if hd < 256 else 0.3
    elements = page * kv_heads * hd
    w = [1 + 0.1 * rng.standard_normal(hd).astype(np.float32) for _ in range(2)]
    steps = [[(0, 50), (1, 7)], [(0, 1), (1, 33), (2, 90)], [(0, 1), (1, 1), (2, 1)], [(2, 1), (0, 20), (1, 1)], [(0, 1), (1, 1), (2, 40)], [(1, 1)]]
    with Buffers(ctx) as b:
        pk, pv = (b.put(np.full((n_pages, elements), NAN[type], np.uint16)) for _ in range(2))
        pw = [b.put(a) for a in w]
        for step in steps:
            entries, seqs, at = [], [], 0
            for s, n in step:
                old = lengths[s]
                lengths[s] += n
                if window:  # the pages that none of this step's rows reaches
                    for i in [i for i in held[s] if (i + 1) * page <= old - window + 1]:
                        free.append(held[s].pop(i))
                        entries.append((s, i, -1))
                for i in range(-(-lengths[s] // page)):
                    if i not in held[s] and i * page >= old - page + 1 and (i + 1) * page > old:
                        held[s][i] = free.pop()
                        entries.append((s, i, held[s][i]))
                seqs.append((at, n, s, lengths[s]))
                at += n
            ctx.page_table_set(table, entries)
            x = rng.standard_normal((at, (heads + 2 * kv_heads) * hd)).astype(np.float32)
            width = x.shape[1]
            shape = ge.heads_shape(F32, type, heads, kv_heads, hd, at, normed=7, q_stride=width, k_stride=width, v_stride=width)
            px, pq, out = b.put(x), b.put(np.zeros((at, heads * hd), np.uint16)), b.put(np.zeros((at, heads * hd), np.uint16))
            ctx.paged_append(shape, rotary, px, px + heads * hd * 4, px + (heads + kv_heads) * hd * 4, pw[0], pw[1], None, table, seqs, pq, pk, pv)
            attention = ge.paged_shape(type, heads, kv_heads, hd, at, scale=scale, window=window, cap=cap)
            ctx.attention_paged(attention, pq, table, pk, pv, seqs, out)
            q = to_float(ctx.download(pq, (at, heads * hd), np.uint16), type).reshape(at, heads, hd)
            got = to_float(ctx.download(out, (at, heads * hd), np.uint16), type).reshape(at, heads, hd)
            pools = [ctx.download(p, (n_pages, kv_heads, page, hd), np.uint16) for p in (pk, pv)]
            for q0, n, s, m in seqs:
                y = x[q0:q0 + n].astype(np.float64).reshape(n, -1, hd)
                rows = [normed(y[:, :heads], w[0].astype(np.float64)), normed(y[:, heads:heads + kv_heads], w[1].astype(np.float64)),
                        normed(y[:, heads + kv_heads:], None)]
                for i in range(2):
                    rows[i], length = turned(rows[i], np.arange(m - n, m), hd)
                    if i == 0:
                        assert (np.abs(q[q0:q0 + n] - rows[0]) <= STEP[type] * np.abs(rows[0]) + 2.0 ** -18 * length + 2.0 ** -25).all()
                # as cached: what the pages hold now
                for j in range(m - n, m):
                    keys[s].append(to_float(pools[0][held[s][j // page], :, j % page], type))
                    values[s].append(to_float(pools[1][held[s][j // page], :, j % page], type))
                k, v = np.stack(keys[s]), np.stack(values[s])
                assert (np.abs(k[m - n:] - rows[1]) <= STEP[type] * np.abs(rows[1]) + 2.0 ** -18 * np.abs(rows[1]).max() + 2.0 ** -25).all()
                assert (np.abs(v[m - n:] - rows[2]) <= STEP[type] * np.abs(rows[2]) + 2.0 ** -18 * np.abs(rows[2]) + 2.0 ** -25).all()
                o, mag = capped_reference(q[q0:q0 + n], k, v, scale, window, cap)
                big = scale * np.sqrt((q[q0:q0 + n] ** 2).sum(-1).max() * (k ** 2).sum(-1).max())
                e = 2 * hd * 2.0 ** -24 * big + cap * 2.0 ** -21
                bound = (STEP[type] + 2 * e + m * 2.0 ** -31) * mag + STEP[type] * np.abs(o) + 1e-7
                assert (np.abs(got[q0:q0 + n] - o) <= bound).all()
                if not window and not cap:
                    flat = ge.attention_shape(type, heads, kv_heads, hd, n, m, scale=scale)
                    fk, fv = (b.put(to_bits(a.reshape(m, -1), type)) for a in (k, v))
                    fo = b.put(np.zeros((n, heads * hd), np.uint16))
                    ctx.attention_causal(flat, pq + q0 * heads * hd * 2, fk, fv, [(0, n, 0, m)], fo)
                    other = to_float(ctx.download(fo, (n, heads * hd), np.uint16), type).reshape(n, heads, hd)
                    assert (np.abs(other - got[q0:q0 + n]) <= 2 * bound).all()
    ctx.rotary_destroy(rotary)
    ctx.page_table_destroy(table)


def test_offsets_past_32_bits(ctx):
    """Pages whose elements lie past 2^32 from the pool's first."""
    kv, hd, page, heads = 1, 128, 256, 2
    stride = (1 << 31) + 64  # elements: 4 GiB a page
    rng = np.random.default_rng(8)
    order, m = [2, 0, 1], 3 * page - 5
    k, v = (to_bits(rng.standard_normal((3 * page, hd)), F16) for _ in range(2))
    x = to_bits(rng.standard_normal((4, (heads + 2) * hd)), F16)
    table = ctx.page_table_create(1, 3, page, 3)
    ctx.page_table_set(table, [(0, i, p) for i, p in enumerate(order)])
    pools = [ctx.alloc(2 * (2 * stride + page * hd)) for _ in range(2)]
    try:
        for pool, a in zip(pools, (k, v)):
            for i, p in enumerate(order):
                ctx.upload(pool + 2 * stride * p, np.ascontiguousarray(a[i * page:(i + 1) * page]))
        with Buffers(ctx) as b:
            px, out = b.put(x), b.put(np.zeros((4, heads * hd), np.uint16))
            width = x.shape[1]
            seqs = [(0, 4, 0, m)]
            heads_shape = ge.heads_shape(F16, F16, heads, kv, hd, 4, q_stride=width, k_stride=width, v_stride=width, page_stride=stride)
            pq = b.put(np.zeros((4, heads * hd), np.uint16))
            ctx.paged_append(heads_shape, None, px, px + heads * hd * 2, px + (heads + 1) * hd * 2, None, None, None, table, seqs, pq, *pools)
            ctx.attention_paged(ge.paged_shape(F16, heads, kv, hd, 4, scale=0.1, page_stride=stride), pq, table, *pools, seqs, out)
            got = to_float(ctx.download(out, (4, heads * hd), np.uint16), F16).reshape(4, heads, hd)
        k[m - 4:m], v[m - 4:m] = x[:, heads * hd:(heads + 1) * hd], x[:, (heads + 1) * hd:]
        o, mag = reference(to_float(x[:, :heads * hd], F16).reshape(4, heads, hd), to_float(k[:m], F16)[:, None], to_float(v[:m], F16)[:, None], 0.1, 0)
        assert (np.abs(got - o) <= 2.0 ** -11 * (mag * 1.01 + np.abs(o)) + 1e-6).all()
    finally:
        for pool in pools:
            ctx.free(pool)
        ctx.page_table_destroy(table)


def test_two_contexts_at_once(ctx):
    """Each with a table and cache of its own, from two threads: the results of one alone."""
    def work(c, seed, out):
        for i in range(6):
            out.append(attend(c, [(0, 30, 400), (30, 1, 900 + i), (31, 1, 77)], 4, 1, 128, F16, seed=seed + i))
            append(c, SEQS, 4, 2, 64, F32, F16, dims=64, normed_heads=7, seed=seed + i)
    alone, both = [], [[], []]
    work(ctx, 40, alone)
    other = ge.Context.create(0)
    errors = []

    def guarded(*a):
        try:
            work(*a)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=guarded, args=(c, 40, o)) for c, o in zip((ctx, other), both)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    other.close()
    assert not errors, errors
    for o in both:
        assert all(np.array_equal(a, b) for a, b in zip(alone, o))
