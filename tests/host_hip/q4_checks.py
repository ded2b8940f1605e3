"""Refusals and clean-up of the 4-bit entries on the host HIP runtime (host_hip.cpp). Run by
tests/test_q4_host.py in a process of its own, whose GE_LIBRARY is the library's objects over that runtime."""
import ctypes as C

import numpy as np
import pytest

import gemma_embed as ge

lib = ge.lib
lib.host_hip_pending.restype = C.c_uint64
lib.host_hip_fail.argtypes = [C.c_char_p, C.c_int]
F32, F16, BF16 = ge.GE_TYPE_F32, ge.GE_TYPE_F16, ge.GE_TYPE_BF16


@pytest.fixture(scope="module")
def ctx():
    c = ge.Context.create(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def memory(ctx):
    return ctx.alloc(1 << 16)


@pytest.fixture
def w(ctx):
    h = ctx.q4_create(np.zeros(18 * 2 * 40, np.uint8), ge.GE_TYPE_Q4_0, 40, 64)
    yield h
    ctx.q4_destroy(h)


@pytest.mark.parametrize("kind,rows,cols", [(ge.GE_TYPE_Q8_0, 4, 64), (F16, 4, 64), (ge.GE_TYPE_Q4_0, 0, 64), (ge.GE_TYPE_Q4_0, -1, 64),
                                            (ge.GE_TYPE_Q4_1, 4, 0), (ge.GE_TYPE_Q4_1, 4, 48)])
def test_refused_matrices(ctx, kind, rows, cols):
    with pytest.raises(ge.GemmaEmbedError) as e:
        ctx.q4_create(np.zeros(4096, np.uint8), kind, rows, cols)
    assert e.value.code == ge.GE_ERR_INVALID


@pytest.mark.parametrize("rows,cols", [((1 << 26) + 1, 32), (1, (1 << 24) + 32)])
def test_matrices_past_the_limits(ctx, rows, cols):
    h = C.c_void_p(1)
    assert lib.ge_op_q4_create(ctx.handle, 16, ge.GE_TYPE_Q4_0, rows, cols, C.byref(h)) == ge.GE_ERR_INVALID and not h.value
    assert lib.ge_op_q4_create(ctx.handle, None, ge.GE_TYPE_Q4_0, 4, 32, C.byref(h)) == ge.GE_ERR_INVALID
    assert lib.ge_op_q4_create(ctx.handle, 16, ge.GE_TYPE_Q4_0, 4, 32, None) == ge.GE_ERR_INVALID


def test_too_few_bytes(ctx):
    with pytest.raises(ge.GemmaEmbedError):
        ctx.q4_create(np.zeros(20 * 8 - 1, np.uint8), ge.GE_TYPE_Q4_1, 4, 64)


def test_refused_products(ctx, memory, w):
    good = (w, memory, F16, 3, memory, F32)
    ctx.gemv_q4(*good)
    for i, bad in ((0, None), (1, None), (1, memory + 4), (2, F32), (2, ge.GE_TYPE_Q4_0), (3, -1), (3, (1 << 19) + 1), (4, None),
                   (4, memory + 2), (5, ge.GE_TYPE_Q8_0)):
        with pytest.raises(ge.GemmaEmbedError) as e:
            ctx.gemv_q4(*(good[:i] + (bad,) + good[i + 1:]))
        assert e.value.code == ge.GE_ERR_INVALID
    ctx.gemv_q4(w, None, F16, 0, None, F32)  # no rows: nothing is read
    assert lib.host_hip_pending() == 0


def test_refused_pairs(ctx, memory, w):
    others = [ctx.q4_create(np.zeros(20 * 2 * 40, np.uint8), ge.GE_TYPE_Q4_1, 40, 64),
              ctx.q4_create(np.zeros(18 * 2 * 41, np.uint8), ge.GE_TYPE_Q4_0, 41, 64),
              ctx.q4_create(np.zeros(18 * 40, np.uint8), ge.GE_TYPE_Q4_0, 40, 32)]
    ctx.gemv_q4_geglu(w, w, memory, BF16, 1, memory, BF16)
    for up in others + [None]:
        for pair in ((w, up), (up, w)):
            with pytest.raises(ge.GemmaEmbedError):
                ctx.gemv_q4_geglu(*pair, memory, BF16, 1, memory, BF16)
    for h in others:
        ctx.q4_destroy(h)


@pytest.mark.parametrize("call,n", [("hipMalloc", 1), ("hipMalloc", 2), ("hipMalloc", 3), ("hipMemcpy", 1), ("hipStreamSynchronize", 1)])
def test_a_failed_creation_gives_no_matrix(ctx, call, n):
    h = C.c_void_p(1)
    blocks = np.zeros(20 * 8, np.uint8)
    lib.host_hip_fail(call.encode(), n)
    assert lib.ge_op_q4_create(ctx.handle, blocks.ctypes.data, ge.GE_TYPE_Q4_1, 4, 64, C.byref(h)) == ge.GE_ERR_GPU
    assert not h.value
    ctx.q4_destroy(ctx.q4_create(blocks, ge.GE_TYPE_Q4_1, 4, 64))
