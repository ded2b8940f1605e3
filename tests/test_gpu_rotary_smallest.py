"""Norms of heads whose elements are fp32's smallest (ge_op_rotate_heads), with no eps that outweighs them, against float64.
The tolerances of test_gpu_rotary.py: squares of elements brought up by 2^90 are 2^-118 on, their mean over up to 512 of them
2^-127, which has 22 bits and so is off by 2^-23 of itself, well within the 16 x 2^-24 of the norm."""
import numpy as np
import pytest

import gemma_embed as ge
from test_gpu_causal import BF16, F16
from test_gpu_rotary import F32, rotate

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("hd", [34, 128, 264, 510, 512])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -149, 2.0 ** -140, 2.0 ** -101])
def test_subnormal_heads(ctx, hd, eps, type):
    def edit(x):
        for t in x:
            tiny = np.float32(2.0 ** -149)
            at = np.arange(t.shape[1])
            t[0] = np.where(at % hd == 1, tiny, 0)                    # one element of a head
            t[1] = np.where(at % 3 == 0, -tiny, tiny)
            t[2] = tiny * np.float32(5) * (at % 7).astype(np.float32)
            t[3] *= np.float32(2.0 ** -126)
            t[4] *= np.float32(2.0 ** -60)
            t[5] *= np.float32(2.0 ** -33)                            # the largest that are brought up
            t[6] *= np.float32(2.0 ** -30)
            t[7, ::2] *= np.float32(2.0 ** -80)
    rotate(ctx, 8, 3, 2, hd, F32, type, dims=hd // 4 * 2, normed_heads=3, edit=edit, eps=eps, seed=hd)


@pytest.mark.parametrize("hd", [128, 510])
def test_subnormal_heads_of_bf16(ctx, hd):
    def edit(x):
        for t in x:
            t[:] = t & 0x8003  # bf16's smallest: up to three times 2^-133
            t[:, ::hd] = 1     # (no head of zeros)
    rotate(ctx, 8, 3, 2, hd, BF16, BF16, dims=hd // 4 * 2, normed_heads=3, edit=edit, eps=0.0, seed=hd)
