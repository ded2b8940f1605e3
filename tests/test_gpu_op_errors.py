"""What a per-op call that failed leaves for the next one."""
import numpy as np
import pytest

import gemma_embed as ge
from test_gpu_causal import F16, attend

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


def test_a_call_after_a_refused_allocation(ctx):
    """Memory that could not be had fails the call that asked for it and no later one."""
    for ask in (lambda: ctx.alloc(1 << 50), lambda: ctx.alloc(1 << 46)):
        with pytest.raises(ge.GemmaEmbedError):
            ask()
        attend(ctx, [(0, 40, 0, 40)], 2, 1, 64, F16)
        w = ctx.q4_create(np.zeros(18 * 4, np.uint8), ge.GE_TYPE_Q4_0, 4, 32)
        ctx.q4_destroy(w)
