"""Limits of a paged cache's entries on the host HIP runtime (host_hip.cpp). Run by tests/test_paged_limits_host.py in a process
of its own, whose GE_LIBRARY is the library's objects over that runtime."""
import numpy as np
import pytest

import gemma_embed as ge
from paged_checks import F16, LAUNCH, ctx, lib, memory, refused  # noqa: F401 (fixtures)


@pytest.mark.parametrize("n", [(1 << 24) - 1, 1 << 24])
def test_sequences_of_an_append(ctx, memory, n):
    """A workgroup each: a launch has under 2^32 threads, which are 2^24 workgroups."""
    h = ctx.page_table_create(n, 1, 8, n)
    entries = np.zeros((n, 3), np.int32)
    entries[:, 0] = entries[:, 2] = np.arange(n)
    ctx.page_table_set(h, entries)
    seqs = np.ones((n, 4), np.uint32)
    seqs[:, 0] = seqs[:, 2] = np.arange(n)
    names = []
    on_launch = LAUNCH(lambda name, args: names.append(name))
    lib.host_hip_on_launch(on_launch)
    try:
        call = (ge.heads_shape(F16, F16, 0, 1, 2, n), None, None, memory, memory, None, None, None, h, seqs, None, memory, memory)
        if n < 1 << 24:
            ctx.paged_append(*call)
        else:
            refused(ctx.paged_append, *call)
    finally:
        lib.host_hip_on_launch(LAUNCH())
    assert len(names) == (n < 1 << 24)
    ctx.page_table_destroy(h)


def test_magnitudes_below_normal_numbers(ctx):
    """A sine or cosine times such a magnitude has few bits: at 2^-147 the products are off by an eighth."""
    for m in (2.0 ** -126, -2.0 ** -126, 0.0, -0.0, 1e-30):
        ctx.rotary_destroy(ctx.rotary_create(64, 1e4, magnitude=m))
    for m in (2.0 ** -127, -2.0 ** -127, 2.0 ** -149):
        refused(ctx.rotary_create, 64, 1e4, magnitude=m)
