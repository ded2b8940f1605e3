"""Attention of causal models (ge_op_attention_causal, ge_op_attention_prefix) against float64.

Tolerance. The inputs are exact. With weights p_j (sum 1), scores off by at most e (fp32 sums of hd products of
magnitude |q||k|: e = scale |q||k| hd 2^-24, times 2 for the softmax's own fp32 steps), weights rounded to the
operands' type (u = 2^-11 or 2^-8 relative, and in fp16 an absolute 2^-25 / 2^6 of the maximum's weight), the
sum of weights exact to fp32, and one rounding of the result:
  |o - o_exact| <= (u + 2 e + n 2^-31) sum_j p_j |v_j| + u |o|, and e itself is below 2^-12 here."""
import numpy as np
import pytest

import gemma_embed as ge

pytestmark = pytest.mark.gpu
F16, BF16 = ge.GE_TYPE_F16, ge.GE_TYPE_BF16
STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8}  # half a step, relative
LAYOUTS = [(2, 1, 64), (6, 2, 64), (4, 4, 128), (3, 1, 256), (2, 1, 512)]


def to_bits(x, kind):
    """float64 -> the type's bits (round to nearest even)."""
    f = np.asarray(x, np.float32)
    if kind == F16:
        return f.astype(np.float16).view(np.uint16)
    b = f.view(np.uint32)
    r = (b + 0x7fff + ((b >> 16) & 1)) >> 16
    return np.where(np.isnan(f), 0x7fc0, r).astype(np.uint16)


def to_float(b, kind):
    if kind == F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


class Buffers:
    """Device copies of arrays, freed together."""

    def __init__(self, ctx):
        self.ctx, self.held = ctx, []

    def put(self, a):
        p = self.ctx.alloc(max(a.nbytes, 16))
        self.held.append(p)
        self.ctx.upload(p, a)
        return p

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for p in self.held:
            self.ctx.free(p)


def reference(q, keys, values, scale, window):
    """(o, sum_j p_j |v_j|) of one sequence in float64: q [n][H][hd], keys and values [m][KV][hd]."""
    n, heads, hd = q.shape
    m, group = len(keys), heads // keys.shape[1]
    o, mag = np.zeros(q.shape), np.zeros(q.shape)
    ahead = np.arange(m)[None, :] - np.arange(n)[:, None] - (m - n)
    hidden = ahead > 0
    if window:
        hidden |= ahead <= -window
    for h in range(heads):
        with np.errstate(all="ignore"):
            s = np.where(hidden, -np.inf, scale * (q[:, h] @ keys[:, h // group].T))
            top = s.max(1, keepdims=True, initial=-np.inf)
            p = np.where(hidden, 0.0, np.exp(s - np.where(top == -np.inf, 0.0, top)))
            p = p / np.where(p.sum(1, keepdims=True) == 0, 1.0, p.sum(1, keepdims=True))
            v = values[:, h // group]
            if np.isfinite(v).all():
                o[:, h], mag[:, h] = p @ v, p @ np.abs(v)
            else:  # hidden values do not count
                for i in range(n):
                    seen = ~hidden[i]
                    o[i, h], mag[i, h] = p[i, seen] @ v[seen], p[i, seen] @ np.abs(v[seen])
    return o, mag


def attend(ctx, seqs, heads, kv_heads, hd, kind, window=0, prefix=0, scale=None, seed=0, pads=(0, 0, 0, 0), spare=3, edit=None,
           values=1.0):
    """One call on random operands, checked against the reference; returns (out bits, the operands)."""
    rng = np.random.default_rng(seed)
    scale = hd ** -0.5 if scale is None else scale
    q_rows = max([s[0] + s[1] for s in seqs] + [0]) + spare
    kv_rows = max([s[2] + s[3] for s in seqs] + [0])
    widths = [heads * hd, kv_heads * hd, kv_heads * hd, heads * hd]
    strides = [w + p for w, p in zip(widths, pads)]

    def rows(n, i, mul=1.0):
        return to_bits(rng.standard_normal((n, strides[i])) * mul, kind)

    t = dict(q=rows(q_rows, 0), k=rows(kv_rows, 1), v=rows(kv_rows, 2, values), pk=rows(prefix, 1), pv=rows(prefix, 2, values))
    if edit:
        edit(t)
    before = rng.integers(0, 1 << 15, (q_rows, strides[3])).astype(np.uint16)
    shape = ge.attention_shape(kind, heads, kv_heads, hd, q_rows, kv_rows, scale=scale, window=window, q_stride=strides[0],
                               k_stride=strides[1], v_stride=strides[2], out_stride=strides[3])
    with Buffers(ctx) as b:
        p = {n: b.put(a) for n, a in t.items()}
        out = b.put(before)
        if prefix:
            ctx.attention_prefix(shape, p["q"], p["pk"], p["pv"], prefix, p["k"], p["v"], seqs, out)
        else:
            ctx.attention_causal(shape, p["q"], p["k"], p["v"], seqs, out)
        got = ctx.download(out, before.shape, np.uint16)
    f = {n: to_float(a, kind) for n, a in t.items()}
    kvw = kv_heads * hd
    want, allowed = {}, {}
    untouched = np.ones(before.shape, bool)
    for i, (q0, n, k0, m) in enumerate(seqs):
        q = f["q"][q0:q0 + n, :heads * hd].reshape(n, heads, hd)
        ks, vs = (np.concatenate([f[a][:, :kvw], f[c][k0:k0 + m, :kvw]]).reshape(-1, kv_heads, hd)
                  for a, c in (("pk", "k"), ("pv", "v")))
        untouched[q0:q0 + n, :heads * hd] = False
        if n == 0:
            continue
        o, mag = reference(q, ks, vs, scale, window)
        with np.errstate(all="ignore"):
            big = abs(scale) * np.sqrt((q ** 2).sum(-1).max() * (ks ** 2).sum(-1).max()) if len(ks) else 0.0
            e = 2 * hd * 2.0 ** -24 * (big if np.isfinite(big) else 1.0)
            u = STEP[kind]
            bound = (u + 2 * e + len(ks) * 2.0 ** -31) * mag + u * np.abs(o) + 1e-7
        y = to_float(got[q0:q0 + n, :heads * hd], kind).reshape(n, heads, hd)
        finite = np.isfinite(o)
        assert np.array_equal(np.isnan(y), np.isnan(o)), f"sequence {i}: NaN in other places"
        assert np.array_equal(y[np.isinf(o)], o[np.isinf(o)]), f"sequence {i}: infinities"
        over = np.abs(y[finite] - o[finite]) - bound[finite]
        assert over.size == 0 or over.max() <= 0, f"sequence {i}: {over.max()} past {bound[finite].max()}"
    assert np.array_equal(got[untouched], before[untouched]), "rows or columns outside the sequences changed"
    return got, t


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("n", [1, 2, 31, 33, 64, 65, 129, 300])
def test_one_prompt(ctx, heads, kv_heads, hd, kind, n):
    attend(ctx, [(0, n, 0, n)], heads, kv_heads, hd, kind, seed=n)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("window", [0, 1, 5, 32, 77])
def test_packed_prompts(ctx, heads, kv_heads, hd, kind, window):
    seqs, at = [], 0
    for n in (7, 0, 1, 150, 32, 63):
        seqs.append((at, n, at, n))
        at += n
    attend(ctx, seqs, heads, kv_heads, hd, kind, window=window, seed=window)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
def test_tokens_over_caches(ctx, heads, kv_heads, hd, kind):
    lengths = [1, 2, 31, 32, 33, 127, 128, 129, 700, 2049]
    seqs, at = [], 0
    for i, n in enumerate(lengths):
        seqs.append((i, 1, at, n))
        at += n + i % 3
    attend(ctx, seqs, heads, kv_heads, hd, kind, seed=1)
    attend(ctx, seqs, heads, kv_heads, hd, kind, seed=1, window=100)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
def test_chunks_over_caches(ctx, heads, kv_heads, hd, kind):
    seqs = [(0, 5, 0, 800), (6, 40, 900, 41), (50, 130, 1000, 1000)]
    attend(ctx, seqs, heads, kv_heads, hd, kind, seed=2)
    attend(ctx, seqs, heads, kv_heads, hd, kind, seed=2, window=200)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("prefix", [1, 63, 64, 1000])
def test_prefix_of_tokens(ctx, heads, kv_heads, hd, kind, prefix):
    attend(ctx, [(i, 1, 5 * i, 1 + i % 5) for i in range(50)], heads, kv_heads, hd, kind, prefix=prefix, seed=prefix)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("window", [0, 3, 90])
def test_prefix_of_texts(ctx, heads, kv_heads, hd, kind, window):
    seqs = [(0, 20, 0, 20), (20, 0, 9, 9), (20, 1, 33, 0), (25, 70, 40, 70), (95, 3, 200, 60), (98, 9, 0, 2)]
    attend(ctx, seqs, heads, kv_heads, hd, kind, window=window, prefix=333, seed=3)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("window", [0, 37, 150])
def test_a_text_behind_a_prefix(ctx, heads, kv_heads, hd, kind, window):
    """Key blocks end at the prefix's last row; NaN and infinities beside the sequence's keys and in values some rows see."""
    def edit(t):
        for row, col in ((80, 0), (99, hd - 1)):
            t["pv"][row, col] = BITS[kind]["nan"]
        t["v"][5, 1], t["v"][120, 0], t["k"][125:] = BITS[kind]["inf"], BITS[kind]["ninf"], BITS[kind]["nan"]
        t["k"][:2] = t["v"][:2] = BITS[kind]["nan"]

    seqs = [(0, 123, 2, 123), (123, 4, 2, 1), (127, 0, 125, 3)]
    attend(ctx, seqs, heads, kv_heads, hd, kind, window=window, prefix=101, seed=21, edit=edit)
    seqs = [(0, 1, 0, 9), (1, 1, 9, 0), (2, 30, 20, 30)]
    attend(ctx, seqs, heads, kv_heads, hd, kind, window=window, prefix=101, seed=22)


@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
def test_queries_before_their_first_key(ctx, heads, kv_heads, hd):
    """Rows that see no key come out as zeros."""
    seqs = [(0, 9, 0, 4), (9, 3, 4, 0), (12, 200, 0, 60)]
    got, _ = attend(ctx, seqs, heads, kv_heads, hd, F16, seed=4)
    assert not got[:5].any() and not got[9:12].any() and not got[12:152].any()
    attend(ctx, [(0, 40, 0, 3)], heads, kv_heads, hd, BF16, prefix=10, seed=4)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("prefix", [0, 50])
def test_strides(ctx, kind, prefix):
    seqs = [(1, 40, 0, 40), (41, 1, 40, 300)]
    for layout in LAYOUTS:
        attend(ctx, seqs, *layout, kind, prefix=prefix, pads=(8, 64, 200, 16), seed=5)


def test_one_projections_output(ctx):
    """q, k and v as views of one buffer's rows."""
    heads, kv_heads, hd, n = 4, 2, 128, 90
    rng = np.random.default_rng(6)
    width = (heads + 2 * kv_heads) * hd
    x = to_bits(rng.standard_normal((n, width)), F16)
    shape = ge.attention_shape(F16, heads, kv_heads, hd, n, n, scale=0.1, q_stride=width, k_stride=width, v_stride=width)
    with Buffers(ctx) as b:
        p, out = b.put(x), b.put(np.zeros((n, heads * hd), np.uint16))
        ctx.attention_causal(shape, p, p + heads * hd * 2, p + (heads + kv_heads) * hd * 2, [(0, n, 0, n)], out)
        got = to_float(ctx.download(out, (n, heads * hd), np.uint16), F16).reshape(n, heads, hd)
    f = to_float(x, F16).reshape(n, -1, hd)
    o, mag = reference(f[:, :heads], f[:, heads:heads + kv_heads], f[:, heads + kv_heads:], 0.1, 0)
    assert (np.abs(got - o) <= 2.0 ** -11 * (mag * 1.01 + np.abs(o)) + 1e-6).all()


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.0, 3.0])
def test_scales(ctx, kind, scale):
    for layout in LAYOUTS:
        attend(ctx, [(0, 70, 0, 70), (70, 1, 0, 200)], *layout, kind, scale=scale, seed=7)
        attend(ctx, [(0, 70, 0, 70)], *layout, kind, scale=scale, prefix=40, seed=7)


BITS = {F16: dict(inf=0x7c00, ninf=0xfc00, nan=0x7e00, low=0xfbff), BF16: dict(inf=0x7f80, ninf=0xff80, nan=0x7fc0, low=0xff7f)}


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
@pytest.mark.parametrize("what", ["inf", "ninf", "nan"])
@pytest.mark.parametrize("window", [0, 20])
def test_non_finite_values_reach_only_the_rows_that_see_them(ctx, heads, kv_heads, hd, kind, what, window):
    def edit(t):
        for row, col in ((3, 0), (50, hd - 1), (99, hd // 2), (99, 1)):
            t["v"][row, col] = BITS[kind][what]

    got, _ = attend(ctx, [(0, 100, 0, 100), (100, 10, 0, 60), (110, 1, 0, 40)], heads, kv_heads, hd, kind, window=window, seed=8,
                    edit=edit)
    first = to_float(got[:99, :heads * hd], kind).reshape(99, heads, hd)
    assert np.isfinite(first[:, :, 1]).all()  # row 99's value is in no earlier row


@pytest.mark.parametrize("kind", [F16, BF16])
def test_infinities_of_both_signs_make_nan(ctx, kind):
    for heads, kv_heads, hd in LAYOUTS:
        def edit(t):
            t["v"][10, 0], t["v"][20, 0] = BITS[kind]["inf"], BITS[kind]["ninf"]

        got, _ = attend(ctx, [(0, 40, 0, 40)], heads, kv_heads, hd, kind, seed=9, edit=edit)
        y = to_float(got[:40, :heads * hd], kind).reshape(40, heads, hd)[:, 0, 0]
        assert np.isfinite(y[:10]).all() and (y[10:20] == np.inf).all() and np.isnan(y[20:]).all()


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("what", ["inf", "ninf", "nan", "low"])
def test_keys_that_no_query_may_see(ctx, kind, what):
    """Anything in the rows behind a sequence and in future keys' scores stays out."""
    for heads, kv_heads, hd in LAYOUTS:
        def edit(t):
            t["k"][40:] = t["v"][40:] = BITS[kind][what]

        attend(ctx, [(0, 40, 0, 40), (50, 3, 20, 20), (53, 0, 90, 4)], heads, kv_heads, hd, kind, seed=10, edit=edit)
        # a future key whose score is not finite
        with Buffers(ctx) as b:
            rng = np.random.default_rng(10)
            q, k, v = (to_bits(rng.standard_normal((40, w * hd)), kind) for w in (heads, kv_heads, kv_heads))
            shape = ge.attention_shape(kind, heads, kv_heads, hd, 40, 40, scale=0.1)
            pq, pv, outs = b.put(q), b.put(v), []
            for bad in (False, True):
                if bad:
                    k[39] = BITS[kind][what]
                out = b.put(np.zeros((40, heads * hd), np.uint16))
                ctx.attention_causal(shape, pq, b.put(k), pv, [(0, 40, 0, 40)], out)
                outs.append(ctx.download(out, (40, heads * hd), np.uint16))
            assert np.array_equal(outs[0][:39], outs[1][:39])


@pytest.mark.parametrize("kind", [F16, BF16])
def test_large_values_and_peaked_scores(ctx, kind):
    for layout in LAYOUTS:
        attend(ctx, [(0, 90, 0, 90), (90, 1, 0, 600)], *layout, kind, scale=1.0, values=100.0, seed=11)


def test_calls_repeat_bitwise_and_ignore_what_ran_before(ctx):
    """The same call gives the same bits, whatever other calls used the temporaries."""
    seqs = [(i, 1, 0, 3000) for i in range(4)]
    one, _ = attend(ctx, seqs, 8, 2, 128, F16, seed=12)
    attend(ctx, [(0, 300, 0, 300)], 3, 1, 256, BF16, prefix=2000, seed=13)
    two, _ = attend(ctx, seqs, 8, 2, 128, F16, seed=12)
    assert np.array_equal(one, two)


def test_neighbours_do_not_change_a_sequence(ctx):
    """A prompt's rows are the same bits alone and in a pack (unsplit calls)."""
    alone, _ = attend(ctx, [(0, 100, 0, 100)], 4, 2, 128, F16, seed=14, spare=100)
    packed, _ = attend(ctx, [(0, 100, 0, 100), (100, 100, 0, 90)], 4, 2, 128, F16, seed=14, spare=0)
    assert np.array_equal(alone[:100], packed[:100])


def test_a_prompt_in_two_chunks_and_token_by_token(ctx):
    """The cache's use: the rows of a prompt computed at once, in chunks and one by one agree."""
    heads, kv_heads, hd, n = 6, 2, 64, 150
    whole, _ = attend(ctx, [(0, n, 0, n)], heads, kv_heads, hd, F16, seed=15)
    chunks, _ = attend(ctx, [(0, 61, 0, 61), (61, n - 61, 0, n)], heads, kv_heads, hd, F16, seed=15)
    tokens, _ = attend(ctx, [(i, 1, 0, i + 1) for i in range(n)], heads, kv_heads, hd, F16, seed=15)
    a, b, c = (to_float(x[:n], F16) for x in (whole, chunks, tokens))
    assert np.abs(a - b).max() <= 4 * 2.0 ** -11 * np.abs(a).max() and np.abs(a - c).max() <= 4 * 2.0 ** -11 * np.abs(a).max()


def test_sequences_share_key_rows(ctx):
    """Several sequences over the same cached rows."""
    for layout in LAYOUTS:
        attend(ctx, [(0, 1, 0, 300), (1, 1, 0, 300), (2, 5, 100, 100), (7, 60, 0, 300)], *layout, F16, seed=16)


@pytest.mark.parametrize("prefix", [0, 40])
def test_offsets_past_32_bits(ctx, prefix):
    """Key rows 4 MiB apart: byte offsets from 4.0 to 4.7 GB, past 2^32 within the sequences."""
    heads, kv_heads, hd, stride, start, n = 2, 1, 64, 1 << 21, 970, 150
    rng = np.random.default_rng(17)
    k, v = (to_bits(rng.standard_normal((start + n, hd)), F16) for _ in range(2))
    pk, pv = (to_bits(rng.standard_normal((prefix, hd)), F16) for _ in range(2))
    q = to_bits(rng.standard_normal((11, heads * hd)), F16)
    shape = ge.attention_shape(F16, heads, kv_heads, hd, 11, start + n, scale=0.125, k_stride=stride, v_stride=stride)
    seqs = [(0, 1, start, n), (1, 10, start + 90, 60)]
    with Buffers(ctx) as b:
        big = [ctx.alloc((start + n) * stride * 2) for _ in range(2)]
        b.held += big
        for p, a in zip(big, (k, v)):
            for r in range(start, start + n):
                ctx.upload(p + r * stride * 2, a[r])
        small = []
        for a in (pk, pv):
            p = ctx.alloc(max(prefix, 1) * stride * 2)
            b.held.append(p)
            for r in range(prefix):
                ctx.upload(p + r * stride * 2, a[r])
            small.append(p)
        out, pq = b.put(np.zeros((11, heads * hd), np.uint16)), b.put(q)
        if prefix:
            ctx.attention_prefix(shape, pq, small[0], small[1], prefix, big[0], big[1], seqs, out)
        else:
            ctx.attention_causal(shape, pq, big[0], big[1], seqs, out)
        got = to_float(ctx.download(out, (11, heads * hd), np.uint16), F16)
    for q0, m, k0, length in seqs:
        ks, vs = (to_float(np.concatenate([x, y[k0:k0 + length]]), F16).reshape(-1, 1, hd) for x, y in ((pk, k), (pv, v)))
        o, mag = reference(to_float(q[q0:q0 + m], F16).reshape(m, heads, hd), ks, vs, 0.125, 0)
        assert (np.abs(got[q0:q0 + m].reshape(m, heads, hd) - o) <= 2.0 ** -11 * (1.01 * mag + np.abs(o)) + 1e-6).all()


def test_two_contexts_at_once():
    """Two threads, a context each, on one GPU: each call gets its own results."""
    import threading
    seqs = [(i, 1, 0, 2000) for i in range(6)]
    first = ge.Context.create(0)
    alone, _ = attend(first, seqs, 8, 2, 128, F16, seed=18, prefix=700)
    other, _ = attend(first, [(0, 200, 0, 200)], 3, 1, 256, BF16, seed=19)
    first.close()
    errors = []

    def run(args, want):
        try:
            c = ge.Context.create(0)
            for _ in range(5):
                got, _ = attend(c, *args[0], **args[1])
                assert np.array_equal(got, want)
            c.close()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    jobs = [(((seqs, 8, 2, 128, F16), dict(seed=18, prefix=700)), alone), ((([(0, 200, 0, 200)], 3, 1, 256, BF16), dict(seed=19)), other)]
    threads = [threading.Thread(target=run, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


def test_bf16_values_near_the_largest(ctx):
    """Sums of weights times values of 1e38 stay inside fp32."""
    for layout in LAYOUTS:
        attend(ctx, [(0, 70, 0, 70), (70, 1, 0, 200)], *layout, BF16, seed=20, values=2.0 ** 124)
