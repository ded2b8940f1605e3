// Norms and rotary positions of query and key heads, and appending keys and values to pages (rotary.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ge {

// Rows [row0, row0 + n) of one sequence, cached at rows first, first + 1, ... of table slot `slot`; workgroups from
// group0 on take rows_each of them each.
struct AppendItem {
    uint32_t row0, n, slot, first, group0;
};
constexpr int kAppendInlineItems = 160;
// The list of a call that has few, among the kernel's arguments.
struct AppendInline {
    AppendItem items[kAppendInlineItems];
};

enum { kNormQ = 1, kNormK = 2, kNormV = 4 };

struct HeadsArgs {
    const void *q, *k, *v;           // rows of heads of the input type; v: appending only
    uint16_t *q_out, *k_out, *v_out;  // k_out and v_out: rows, or pages when appending
    const float *q_norm, *k_norm;    // [head_dim], null: no weight
    const int32_t* positions;        // [rows], null: the cache row (appending only)
    const double* turns;             // [half]: turns of a full circle a position
    const int32_t* table;            // [slots][slot_pages]
    const AppendItem* items;         // appending: an item a workgroup; null: in AppendInline, to be searched
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // elements from one row to the next
    int64_t page_stride;             // elements from one page to the next
    int heads, kv_heads, head_dim, rows;
    int half;                        // pairs that turn, from the first element on
    int pairs;                       // 1: neighbours are a pair, 0: elements half apart
    int normed;                      // kNorm bits
    float eps, fade, gain;           // fade gain: the magnitude, fade <= 1 <= |gain|
    int rows_each, workgroups;       // rows of a workgroup
    int n_items, slot_pages, page_shift;
};
static_assert(sizeof(HeadsArgs) + sizeof(AppendInline) <= 4096, "kernel arguments");

// Rows of a workgroup. Few rows: one, its heads shared out to the waves, which then are one step long (to append 60,
// 300, 1000, 2048 and 4000 tokens of 32 + 8 + 8 heads of 128: 6.0, 6.7, 9.8, 18.5 and 35 us, with a row a wave 10.7, 10.7, 12.5, 18.0
// and 26). Else a row a wave, up to 4096 workgroups (16384 rows of 32 + 8 heads of 128 in 4096, 2048, 1024 and 512: 66.7, 70.9,
// 73.5 and 83.0 us).
inline int heads_rows_each(int rows) { return rows <= 1024 ? 1 : rows <= 4 * 4096 ? 4 : (rows / 4096 + 3) / 4 * 4; }

// Whether heads and the pairs that turn come in units of 8, 4, 2 or 1 elements, of which a wave holds 64 of each half of a
// head (units of 1: four a lane).
inline bool heads_unit_ok(int head_dim, int half, int unit) {
    return unit == 1 || ((unit == 2 || unit == 4 || unit == 8) && head_dim % (2 * unit) == 0 && head_dim <= 128 * unit && half % unit == 0);
}

// unit: one for which heads_unit_ok holds and in which every stride and every address come (fp32 rows: 16 bytes at most).
hipError_t launch_rotate_heads(hipStream_t s, const HeadsArgs& a, bool in_f32, bool bf16, int unit);
hipError_t launch_append(hipStream_t s, const HeadsArgs& a, const AppendInline& in, bool in_f32, bool bf16, int unit);
// Page numbers into a table: entries of (place in the table, page) pairs.
hipError_t launch_table_set(hipStream_t s, int32_t* table, const uint2* entries, int n);

}  // namespace ge
