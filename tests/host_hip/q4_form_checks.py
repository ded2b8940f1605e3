"""Which launch form a 4-bit product takes at the sizes of tests/q4_forms.py, on the host HIP runtime
(host_hip.cpp). Run by tests/test_q4_forms_host.py in a process of its own, whose GE_LIBRARY is the library's
objects over that runtime."""
import ctypes as C
import os
import re
import sys

import numpy as np
import pytest

import gemma_embed as ge

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from q4_forms import FORMS, NEIGHBOURS  # noqa: E402

LAUNCH = C.CFUNCTYPE(None, C.c_char_p, C.POINTER(C.c_void_p))
lib = ge.lib
lib.host_hip_on_launch.argtypes = [LAUNCH]


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


def form(ctx, m, rows, cols, geglu, kind=ge.GE_TYPE_Q4_0):
    """The kernel of a product: (16-row tiles of x, accumulator registers, row blocks, x in LDS), matrices, minima."""
    bytes_ = 20 if kind == ge.GE_TYPE_Q4_1 else 18
    w, memory, names = ctx.q4_create(np.zeros(rows * cols // 32 * bytes_, np.uint8), kind, rows, cols), ctx.alloc(16), []
    callback = LAUNCH(lambda name, args: names.append(name.decode()))
    lib.host_hip_on_launch(callback)
    try:
        if geglu:
            ctx.gemv_q4_geglu(w, w, memory, ge.GE_TYPE_F16, m, memory, ge.GE_TYPE_F16)
        else:
            ctx.gemv_q4(w, memory, ge.GE_TYPE_F16, m, memory, ge.GE_TYPE_F16)
    finally:
        lib.host_hip_on_launch(LAUNCH())
        ctx.q4_destroy(w)
        ctx.free(memory)
    assert len(names) == 1
    nt, mr, rb, mats, least, lds = map(int, re.search(r"gemv_q4_kernelI.*?Li(\d)ELi(\d)ELi(\d)ELi(\d)ELb(\d)ELb(\d)E", names[0]).groups())
    return (nt, mr, rb, bool(lds)), mats, bool(least)


@pytest.mark.parametrize("kind", [ge.GE_TYPE_Q4_0, ge.GE_TYPE_Q4_1])
@pytest.mark.parametrize("m,rows,cols,geglu,want", FORMS)
def test_form(ctx, m, rows, cols, geglu, want, kind):
    got, mats, least = form(ctx, m, rows, cols, geglu, kind)
    assert got == want and mats == (2 if geglu else 1) and least == (kind == ge.GE_TYPE_Q4_1)


def test_every_form_is_among_them():
    plain = {want for *_, geglu, want in FORMS if not geglu}
    assert plain == {(1, 1, 1, True), (1, 2, 1, False)} | {(nt, 4, rb, False) for nt in (1, 2, 4) for rb in (1, 2)} | {(1, 4, 4, False)}


def test_the_neighbours_take_different_forms(ctx):
    rows, cols, counts = NEIGHBOURS
    assert len({form(ctx, m, rows, cols, False)[0] for m in counts}) == 5
