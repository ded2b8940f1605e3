"""Calls of attention over a shared prefix whose texts stack up over it, for the host check that they do and the
GPU tests that compare them with float64: (name, heads, KV heads, head dim, prefix, sequences)."""


def _texts(lengths, own=None):
    """Texts of these many tokens back to back; own keys: as many, or those of own(i, n)."""
    out, q, kv = [], 0, 0
    for i, n in enumerate(lengths):
        m = n if own is None else own(i, n)
        out.append((q, n, kv, m))
        q += n
        kv += m
    return out


def _calls():
    out = []
    for heads, kv_heads, hd, prefix in ((2, 1, 64, 6000), (6, 2, 64, 3001), (4, 4, 128, 1500), (3, 1, 256, 2000), (2, 1, 512, 1100)):
        layout = (heads, kv_heads, hd, prefix)
        out += [
            # single tokens, over the prefix and up to four rows of their own
            ("tokens",) + layout + (_texts([1] * 200, lambda i, n: 1 + i % 5),),
            # no own keys: the prefix's part is the result
            ("alone",) + layout + (_texts([1] * 200, lambda i, n: 0),),
            # some with none, some whose first token sees the prefix only
            ("mixed",) + layout + (_texts([1 + i % 3 for i in range(160)], lambda i, n: n - 1 + i % 2),),
            # short texts, a longer cache among them
            ("texts",) + layout + (_texts([1 + 2 * (i % 4) for i in range(300)], lambda i, n: n + 300 * (i == 20)),),
            # a run that stacks between texts that do not: unused rows, and a query that sees no whole prefix
            ("apart",) + layout + ([(0, 9, 0, 2)] + [(9 + q, n, 2 + k, m) for q, n, k, m in _texts([2] * 150)] + [(320, 5, 0, 5)],),
        ]
    # more keys than one part of a tile takes
    out.append(("split", 8, 2, 128, 9000, _texts([1] * 64, lambda i, n: 2 + i % 9)))
    out.append(("split", 3, 1, 256, 8192, _texts([8 + 5 * (i % 9) for i in range(64)])))
    return out


STACKED = _calls()
