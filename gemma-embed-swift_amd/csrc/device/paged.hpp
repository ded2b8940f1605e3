// Attention over pages of keys and values (paged.hip).
#pragma once

#include "causal.hpp"

namespace ge {

// k and v are pools of pages, page p at p page_stride: [kv_heads][1 << page_shift rows][head_dim]. Key j of slot s
// is row j mod the page's rows of page table[s slot_pages + (j >> page_shift)]; an item's key0 is its slot and its
// k_lo a multiple of kPagedAlign.
struct PagedArgs : CausalArgs {
    const int32_t* table;
    int64_t page_stride;
    int slot_pages, page_shift;
    // Scores x (q k unscaled) capped: cap_top tanh(cap_z x), in log2; c is then 1. 0: as they are.
    float cap_z, cap_top;
    uint32_t cap_fine;  // also where the argument is small
};
static_assert(sizeof(PagedArgs) + sizeof(CausalInline) <= 4096, "kernel arguments");

constexpr int kPagedAlign = 8;  // copies are of 8 keys, which are in one page

// Head dims as causal_head_dim_ok; kinds: the CausalKind of the items. Joins: launch_causal_join.
hipError_t launch_paged(hipStream_t s, const PagedArgs& a, const CausalInline& in, int hd, bool bf16, int kinds);
// Dynamic LDS limits; once per device, before launching.
hipError_t paged_configure();

}  // namespace ge
