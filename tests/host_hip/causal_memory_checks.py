"""What a context keeps of a call's work lists, on the host HIP runtime (host_hip.cpp). Run by
tests/test_causal_memory.py in a process of its own, whose GE_LIBRARY is the library's objects over that runtime."""
import ctypes as C
import os
import sys

import numpy as np
import pytest

import gemma_embed as ge

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from causal_checks import LAUNCH, Args, P, lib  # noqa: E402

KEPT = 16 << 20


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


def block(p):
    """Bytes of the allocation that holds p, None if there is none."""
    base, size = P(), C.c_size_t()
    return size.value if lib.host_hip_block(P(p), C.byref(base), C.byref(size)) else None


def lists(ctx, n, fail=None):
    """One token of each of n texts over its one key: the lists' place, and their allocation during the call."""
    memory = ctx.alloc(1 << 12)
    seqs = np.zeros((n, 4), np.uint32)
    seqs[:, 0], seqs[:, 1], seqs[:, 3] = np.arange(n), 1, 1
    seen = []

    def on_launch(name, args):
        at = C.cast(C.cast(args[0], C.POINTER(Args))[0].items, P).value
        seen.append((at, block(at)))
    callback = LAUNCH(on_launch)
    lib.host_hip_on_launch(callback)
    if fail:
        lib.host_hip_fail(fail.encode(), 1)
    try:
        ctx.attention_causal(ge.attention_shape(ge.GE_TYPE_F16, 1, 1, 64, n, 1), memory, memory, memory, seqs, memory)
    finally:
        lib.host_hip_on_launch(LAUNCH())
        ctx.free(memory)
        lists.seen = seen
    assert len(seen) == 1
    return seen[0]


def test_small_lists_stay_for_the_next_call(ctx):
    at, size = lists(ctx, 1000)
    assert 36000 <= size <= KEPT and block(at) == size
    assert lists(ctx, 900) == (at, size)


@pytest.mark.parametrize("fail", [None, "hipStreamSynchronize"])
def test_large_lists_are_given_back(ctx, fail):
    if fail:
        with pytest.raises(ge.GemmaEmbedError):
            lists(ctx, 500000, fail)
    else:
        lists(ctx, 500000)
    at, size = lists.seen[0]
    assert size >= 500000 * 36 and block(at) is None
    small = lists(ctx, 1000)
    assert small[1] <= KEPT and block(small[0])
