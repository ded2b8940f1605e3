// Attention of causal models (causal.hip): the items the host plans (causal.cpp) and the kernels take.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ge {

// Items by the stacked rows they take: wide ones share each key block between the waves' rows, narrow ones
// have up to 32 rows and a key block a wave.
enum CausalKind { kCausalWide = 1, kCausalNarrow = 2 };
constexpr int causal_wide_rows(int hd) { return hd > 256 ? 64 : 128; }
constexpr int kCausalNarrowRows = 32;
constexpr uint32_t kDirect = 0xffffffffu;
// Workgroups of a launch: HIP's grid counts work-items in 32 bits.
constexpr uint64_t kCausalMaxGroups = (uint64_t(1) << 32) / 256 - 1;

// Stacked rows [row0, row0 + n_rows) (token row / group from q_token on) against the keys [k_lo, k_hi). A
// sequence's keys count through: the prefix's rows are 0 .. prefix_len - 1, its own, from row key0 of k and v on,
// prefix_len and up. Row token i sees key j iff j <= i + shift and, with a window, j > i + shift - window.
struct CausalItem {
    uint32_t q_token, row0, n_rows;
    uint32_t key0, k_lo, k_hi;
    int32_t shift;
    uint32_t part;  // kDirect: the rows go to out; else to the partial rows from here on
    uint32_t narrow;
};

// Rows [row0, row0 + n_rows) of q_token's sequence joined from splits[0] parts at partial rows
// part[0] + s stride[0] and splits[1] parts at part[1] + s stride[1].
struct CausalJoin {
    uint32_t q_token, row0, n_rows;
    uint32_t part[2], stride[2], splits[2];
};

struct CausalArgs {
    const uint16_t *q, *k, *v, *prefix_k, *prefix_v;
    uint16_t* out;
    const CausalItem* items;  // null: in CausalInline, as the joins
    const CausalJoin* joins;
    float* part_o;    // fp32 [kv_heads][part_rows][head_dim], unnormalised
    float2* part_ml;  // [kv_heads][part_rows]: running maximum (log2) and sum
    int64_t q_stride, k_stride, v_stride, out_stride;  // elements from one row to the next
    size_t part_rows;
    int n_items, n_joins;
    int join_rows;  // the most rows of a join
    int group, kv_heads, window;  // window 0: none
    int prefix_len;
    float c;                      // |scale| log2(e)
    uint32_t q_flip;              // the sign bits of two values where the scale is negative
};

// The lists of a call that has few of both, among the kernel's arguments: a workgroup finds its item with
// them instead of after a second read over the bus.
constexpr int kCausalInlineItems = 48, kCausalInlineJoins = 40;
struct CausalInline {
    CausalItem items[kCausalInlineItems];
    CausalJoin joins[kCausalInlineJoins];
};
static_assert(sizeof(CausalArgs) + sizeof(CausalInline) <= 4096, "kernel arguments");

// Head dims 64, 128, 256 and 512.
bool causal_head_dim_ok(int hd);
// kinds: the CausalKind of the items.
hipError_t launch_causal(hipStream_t s, const CausalArgs& a, const CausalInline& in, int hd, bool bf16, int kinds);
hipError_t launch_causal_join(hipStream_t s, const CausalArgs& a, const CausalInline& in, int hd, bool bf16);
// Dynamic LDS limits; once per device, before launching (24 kernels: 2 ms of a context's creation otherwise).
hipError_t causal_configure();

}  // namespace ge
