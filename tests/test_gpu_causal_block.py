"""The operators of causal models together, as a decoder layer of 4-bit weights uses them: a prompt through the
projections, the attention and the feed-forward, then the next tokens of a batch over the prompt's keys. Every
step is compared with float64 on the inputs it really had (the step before it, as stored), so each has its own
operator's tolerance: half a step of fp16 of the result and of what the softmax weights multiply, and fp32 sums."""
import math

import numpy as np
import pytest

import gemma_embed as ge

pytestmark = pytest.mark.gpu
F16, F32, Q4 = ge.GE_TYPE_F16, ge.GE_TYPE_F32, ge.GE_TYPE_Q4_0
H, KV, HD, D, FF = 6, 2, 64, 256, 352
WIDTH = (H + 2 * KV) * HD
HALF = 2.0 ** -11


def weights(rng, rows, cols):
    q = rng.integers(0, 16, (rows * cols // 32, 32))
    d = (np.abs(rng.standard_normal(len(q))) * 0.01 + 0.005).astype(np.float16)
    blocks = np.concatenate([d.view(np.uint8).reshape(-1, 2), (q[:, :16] | q[:, 16:] << 4).astype(np.uint8)], 1)
    return blocks, (d.astype(np.float64)[:, None] * (q - 8)).reshape(rows, cols)


def attention(q, k, v):
    """[n][H][HD] over the last of [m][KV][HD], and what each weight multiplies."""
    n, m, o, mag = len(q), len(k), np.zeros(q.shape), np.zeros(q.shape)
    hidden = np.arange(m)[None, :] > np.arange(n)[:, None] + m - n
    for h in range(H):
        s = np.where(hidden, -np.inf, q[:, h] @ k[:, h * KV // H].T * HD ** -0.5)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        o[:, h], mag[:, h] = p @ v[:, h * KV // H], p @ np.abs(v[:, h * KV // H])
    return o, mag


def gelu(x):
    return 0.5 * x * (1 + np.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))


class Layer:
    def __init__(self, ctx, rng):
        self.ctx, self.held = ctx, []
        shapes = dict(qkv=(WIDTH, D), o=(D, H * HD), gate=(FF, D), up=(FF, D))
        self.w, self.handle = {}, {}
        for name, (rows, cols) in shapes.items():
            blocks, self.w[name] = weights(rng, rows, cols)
            self.handle[name] = ctx.q4_create(blocks, Q4, rows, cols)

    def put(self, a):
        p = self.ctx.alloc(a.nbytes)
        self.held.append(p)
        self.ctx.upload(p, a)
        return p

    def half(self, p, shape):
        return self.ctx.download(p, shape, np.float16).astype(np.float64)

    def close(self):
        for p in self.held:
            self.ctx.free(p)
        for h in self.handle.values():
            self.ctx.q4_destroy(h)

    def projection(self, name, x, px, kind=F16):
        """x W^T on the device (rows of kind), checked; x: the values at px."""
        n, rows = len(x), len(self.w[name])
        p = self.put(np.zeros((n, rows), np.float16 if kind == F16 else np.float32))
        self.ctx.gemv_q4(self.handle[name], px, F16, n, p, kind)
        got = self.ctx.download(p, (n, rows), np.float16 if kind == F16 else np.float32).astype(np.float64)
        want, size = x @ self.w[name].T, np.abs(x) @ np.abs(self.w[name]).T
        steps = (HALF if kind == F16 else 2.0 ** -24) * np.abs(want)
        assert (np.abs(got - want) <= steps * 1.01 + 60 * 2.0 ** -24 * 16 * size + 1e-7).all(), name
        return p, got

    def feed_forward(self, x, px):
        n = len(x)
        p = self.put(np.zeros((n, FF), np.float16))
        self.ctx.gemv_q4_geglu(self.handle["gate"], self.handle["up"], px, F16, n, p, F16)
        got, g, u = self.half(p, (n, FF)), x @ self.w["gate"].T, x @ self.w["up"].T
        want = gelu(g) * u
        size = np.abs(x) @ np.abs(self.w["gate"]).T * (np.abs(u) + 1) + np.abs(x) @ np.abs(self.w["up"]).T * (np.abs(g) + 1)
        assert (np.abs(got - want) <= HALF * 1.01 * np.abs(want) + 60 * 2.0 ** -24 * 16 * size + 1e-6).all()


def test_a_layer_over_a_prompt_and_the_next_tokens():
    rng, ctx = np.random.default_rng(1), ge.Context.create(0)
    layer, prompt, batch = Layer(ctx, rng), 45, 9
    try:
        x = rng.standard_normal((prompt, D)).astype(np.float16)
        px = layer.put(x)
        p_qkv, qkv = layer.projection("qkv", x.astype(np.float64), px)
        parts = qkv.reshape(prompt, -1, HD)
        # the prompt's attention reads q, k and v where the projection left them
        shape = ge.attention_shape(F16, H, KV, HD, prompt, prompt, scale=HD ** -0.5, q_stride=WIDTH, k_stride=WIDTH, v_stride=WIDTH)
        p_attn = layer.put(np.zeros((prompt, H * HD), np.float16))
        ctx.attention_causal(shape, p_qkv, p_qkv + H * HD * 2, p_qkv + (H + KV) * HD * 2, [(0, prompt, 0, prompt)], p_attn)
        attn = layer.half(p_attn, (prompt, H, HD))
        o, mag = attention(parts[:, :H], parts[:, H:H + KV], parts[:, H + KV:])
        assert (np.abs(attn - o) <= HALF * 1.02 * (mag + np.abs(o)) + 1e-6).all()
        layer.projection("o", attn.reshape(prompt, -1), p_attn, F32)
        layer.feed_forward(x.astype(np.float64), px)

        # one more token of each text of a batch, over the prompt's keys and its own
        y = rng.standard_normal((batch, D)).astype(np.float16)
        py = layer.put(y)
        p_new, new = layer.projection("qkv", y.astype(np.float64), py)
        tokens = new.reshape(batch, -1, HD)
        step = ge.attention_shape(F16, H, KV, HD, batch, batch, scale=HD ** -0.5, q_stride=WIDTH, k_stride=WIDTH, v_stride=WIDTH)
        p_step = layer.put(np.zeros((batch, H * HD), np.float16))
        seqs = [(i, 1, i, 1) for i in range(batch)]
        ctx.attention_prefix(step, p_new, p_qkv + H * HD * 2, p_qkv + (H + KV) * HD * 2, prompt, p_new + H * HD * 2,
                             p_new + (H + KV) * HD * 2, seqs, p_step)
        got = layer.half(p_step, (batch, H, HD))
        for i in range(batch):
            k, v = (np.concatenate([parts[:, a:a + KV], tokens[i:i + 1, a:a + KV]]) for a in (H, H + KV))
            o, mag = attention(tokens[i:i + 1, :H], k, v)
            assert (np.abs(got[i:i + 1] - o) <= HALF * 1.02 * (mag + np.abs(o)) + 1e-6).all(), i
        layer.projection("o", got.reshape(batch, -1), p_step, F32)
        layer.feed_forward(y.astype(np.float64), py)

        # the same tokens over caches of their own: the prompt's rows and one more each, copied together
        cache = np.zeros((batch, prompt + 1, 2 * KV * HD), np.float16)
        cache[:, :prompt] = qkv[:, H * HD:]
        cache[:, prompt] = new[:, H * HD:]
        p_cache = layer.put(cache)
        own = ge.attention_shape(F16, H, KV, HD, batch, batch * (prompt + 1), scale=HD ** -0.5, q_stride=WIDTH,
                                 k_stride=2 * KV * HD, v_stride=2 * KV * HD)
        p_own = layer.put(np.zeros((batch, H * HD), np.float16))
        ctx.attention_causal(own, p_new, p_cache, p_cache + KV * HD * 2, [(i, 1, i * (prompt + 1), prompt + 1) for i in range(batch)], p_own)
        assert np.abs(layer.half(p_own, (batch, H, HD)) - got).max() <= 4 * HALF * np.abs(got).max()
    finally:
        layer.close()
        ctx.close()
