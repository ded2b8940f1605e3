"""Infinite values behind keys that weigh nothing (ge_op_attention_causal, ge_op_attention_prefix), in parts of a row of their
own: 0 times infinity in the definition. Against float64, with the tolerances of test_gpu_causal.py."""
import numpy as np
import pytest

import gemma_embed as ge
from test_gpu_causal import BF16, attend, to_bits, to_float

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.mark.parametrize("heads,kv_heads,hd", [(2, 1, 64), (4, 4, 128), (3, 1, 256), (2, 1, 512)])
@pytest.mark.parametrize("prefix", [0, 1500])
def test_infinite_values_of_keys_that_weigh_nothing(ctx, heads, kv_heads, hd, prefix):
    def edit(t):
        t["q"][:] = to_bits(np.full(t["q"].shape, 2.0 ** 40), BF16)
        k, v = (t["pk"], t["pv"]) if prefix else (t["k"], t["v"])
        k[:1024] = to_bits(np.full((1024, k.shape[1]), -(2.0 ** 100)), BF16)
        v[5, 3] = 0x7f80
        v[70, -1] = 0x7fc0
        v[1400, 9] = 0x7f80

    got, _ = attend(ctx, [(0, 1, 0, 4000)], heads, kv_heads, hd, BF16, prefix=prefix, scale=2.0 ** -44, edit=edit, seed=hd)
    f = to_float(got[0], BF16).reshape(heads, hd)
    assert np.isnan(f[0, 3]) and np.isnan(f[-1, hd - 1]) and f[0, 9] == np.inf and np.isfinite(f[0, 4:9]).all()
