"""The 4-bit products in every launch form (tests/q4_forms.py) against float64, with the tolerances of
test_gpu_q4.py."""
import numpy as np
import pytest

import gemma_embed as ge
from q4_forms import FORMS, NEIGHBOURS
from test_gpu_q4 import BF16, F16, F32, TYPES, check, matrix, to_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("x_kind", [F16, BF16])
@pytest.mark.parametrize("m,rows,cols,geglu,form", FORMS)
def test_forms(ctx, m, rows, cols, geglu, form, kind, x_kind):
    check(ctx, kind, m, rows, cols, x_kind, F32, geglu=geglu, seed=m)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("x_kind", [F16, BF16])
@pytest.mark.parametrize("geglu", [False, True])
def test_a_rows_bits_in_every_form(ctx, kind, x_kind, geglu):
    rows, cols, counts = NEIGHBOURS
    rng = np.random.default_rng(7)
    x = to_bits(rng.standard_normal((max(counts), cols)), x_kind)
    w = [ctx.q4_create(matrix(rng, kind, rows, cols)[0], kind, rows, cols) for _ in range(1 + geglu)]
    px, py, got = ctx.alloc(x.nbytes), ctx.alloc(len(x) * rows * 4), {}
    ctx.upload(px, x)
    for m in counts:
        (ctx.gemv_q4_geglu if geglu else ctx.gemv_q4)(*w, px, x_kind, m, py, F32)
        got[m] = ctx.download(py, (m, rows), np.uint32)
    ctx.free(px), ctx.free(py)
    for h in w:
        ctx.q4_destroy(h)
    for m in counts:
        assert np.array_equal(got[m], got[max(counts)][:m]), m
