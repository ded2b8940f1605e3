// Per-op entries of 4-bit weights (ge_op_q4_create, ge_op_gemv_q4, ge_op_gemv_q4_geglu).
#include <hip/hip_runtime.h>

#include <memory>

#include "q4.hpp"
#include "runtime_internal.hpp"

struct ge_q4_matrix {
    ge::Q4Dev m;
};

namespace ge {
namespace {

void free_planes(Q4Dev& w) {
    if (w.q) (void)hipFree(w.q);
    if (w.d) (void)hipFree(w.d);
    if (w.m) (void)hipFree(w.m);
    w = Q4Dev{};
}

void product(ge_ctx* c, const ge_q4_matrix* w, const ge_q4_matrix* up, const void* x, int32_t x_type, int32_t rows, void* y,
             int32_t y_type) {
    if (!w) fail(GE_ERR_INVALID, "null matrix");
    if (up && (up->m.rows != w->m.rows || up->m.cols != w->m.cols || !up->m.m != !w->m.m))
        fail(GE_ERR_INVALID, "gate and up must have the same shape and type");
    if (x_type != GE_TYPE_F16 && x_type != GE_TYPE_BF16) fail(GE_ERR_INVALID, "4-bit product: x of type %d (F16 or BF16)", x_type);
    if (y_type != GE_TYPE_F32 && y_type != GE_TYPE_F16 && y_type != GE_TYPE_BF16)
        fail(GE_ERR_INVALID, "4-bit product: y of type %d (F32, F16 or BF16)", y_type);
    if (rows < 0 || rows > kQ4MaxRows) fail(GE_ERR_INVALID, "4-bit product: %d rows (0 to %d)", rows, kQ4MaxRows);
    if (rows == 0) return;
    if (!x || !y || reinterpret_cast<uintptr_t>(x) % 16 || reinterpret_cast<uintptr_t>(y) % 16)
        fail(GE_ERR_INVALID, "4-bit product: x and y, 16-byte aligned");
    Q4Args a{w->m, up ? up->m : Q4Dev{}, static_cast<const uint16_t*>(x), y, rows};
    const Q4Out out = y_type == GE_TYPE_F32 ? kQ4F32 : y_type == GE_TYPE_F16 ? kQ4F16 : kQ4BF16;
    launch(c, up ? "gemv_q4_geglu" : "gemv_q4",
           [&] { return launch_gemv_q4(c->stream, a, x_type == GE_TYPE_BF16, up != nullptr, out); });
    hip_check(hipStreamSynchronize(c->stream), "hipStreamSynchronize");
}

}  // namespace
}  // namespace ge

using ge::fail;
using ge::guarded;

extern "C" {

int ge_op_q4_create(ge_ctx* c, const void* q4_rows, int32_t type, int32_t rows, int32_t cols, ge_q4_matrix** out) {
    if (out) *out = nullptr;
    ge::Q4Dev w;
    void* raw = nullptr;
    const int rc = guarded(c, [&] {
        if (type != GE_TYPE_Q4_0 && type != GE_TYPE_Q4_1) fail(GE_ERR_INVALID, "4-bit matrix of type %d (Q4_0 or Q4_1)", type);
        if (!q4_rows || !out || rows <= 0 || cols <= 0 || cols % 32)
            fail(GE_ERR_INVALID, "4-bit matrix needs rows > 0 and cols a multiple of 32");
        if (rows > ge::kQ4MaxWeightRows || cols > ge::kQ4MaxCols)
            fail(GE_ERR_INVALID, "4-bit matrix of %d x %d (up to %d x %d)", rows, cols, ge::kQ4MaxWeightRows, ge::kQ4MaxCols);
        std::unique_ptr<ge_q4_matrix> m(new ge_q4_matrix);
        w.rows = rows;
        w.cols = cols;
        w.tiles = ge::q4_tiles(cols);
        const size_t tiles = size_t(ge::q4_row_blocks(rows)) * size_t(w.tiles);
        const size_t bytes = size_t(rows) * size_t(cols / 32) * (type == GE_TYPE_Q4_1 ? 20 : 18);
        raw = ge::dev_alloc(bytes, "4-bit matrix");
        w.q = static_cast<uint32_t*>(ge::dev_alloc(tiles * 1024, "4-bit matrix"));
        w.d = static_cast<uint16_t*>(ge::dev_alloc(tiles * 128, "4-bit matrix"));
        if (type == GE_TYPE_Q4_1) w.m = static_cast<uint16_t*>(ge::dev_alloc(tiles * 128, "4-bit matrix"));
        ge::hip_check(hipMemcpy(raw, q4_rows, bytes, hipMemcpyHostToDevice), "hipMemcpy");
        ge::launch(c, "q4_repack", [&] { return ge::launch_q4_repack(c->stream, static_cast<const unsigned char*>(raw), w); });
        ge::hip_check(hipStreamSynchronize(c->stream), "hipStreamSynchronize");
        m->m = w;
        *out = m.release();
    });
    if (raw) (void)hipFree(raw);
    if (rc != GE_OK) ge::free_planes(w);
    return rc;
}

int ge_op_q4_destroy(ge_ctx* c, ge_q4_matrix* m) {
    if (!m) return GE_OK;
    const int rc = guarded(c, [&] { ge::free_planes(m->m); });
    delete m;
    return rc;
}

int ge_op_gemv_q4(ge_ctx* c, const ge_q4_matrix* w, const void* x, int32_t x_type, int32_t m, void* y, int32_t y_type) {
    return guarded(c, [&] { ge::product(c, w, nullptr, x, x_type, m, y, y_type); });
}

int ge_op_gemv_q4_geglu(ge_ctx* c, const ge_q4_matrix* gate, const ge_q4_matrix* up, const void* x, int32_t x_type, int32_t m,
                        void* act, int32_t act_type) {
    return guarded(c, [&] {
        if (!up) fail(GE_ERR_INVALID, "null matrix");
        ge::product(c, gate, up, x, x_type, m, act, act_type);
    });
}

}  // extern "C"
