"""Calls of attention over pages (ge_op_attention_paged) in which a workgroup takes several items, one after another:
many single tokens, or these with chunks among them, over so many KV heads that few workgroups a head run at once. And
calls that end in more joins than fit among a launch's arguments. The host checks show that they are planned so, the GPU
tests what comes out."""

# heads, KV heads, head dim: eight workgroups a KV head run at once
LAYOUTS = [(128, 128, 64), (256, 128, 64), (64, 64, 128), (128, 64, 128), (64, 64, 256), (32, 32, 512), (64, 32, 512)]
# few KV heads
JOINED = [(4, 1, 64), (2, 1, 128), (2, 1, 256), (4, 4, 512), (2, 2, 512)]
WINDOW = 200


def placed(lengths):
    """(q_start, q_len, kv_len) of rows back to back, from (q_len, kv_len)."""
    out, at = [], 0
    for n, m in lengths:
        out.append((at, n, m))
        at += n
    return out


def tokens():
    return placed([(1, 130 + 37 * i % 401) for i in range(44)])


def mixed(n, every, chunk):
    """Single tokens, and every so many a chunk of `chunk` rows or of 3."""
    return placed([((chunk if i % (2 * every) else 3) if i % every == 0 else 1, 130 + 37 * i % 380) for i in range(n)])


def joined():
    return placed([(1, 200 + 13 * i) for i in range(60)])


# the second's 60 to 90 items lie among a launch's arguments, the third's more than 90 in a list in memory
CALLS = {"tokens": tokens(), "chunks among them": mixed(60, 5, 50), "a list of items": mixed(90, 10, 33)}
