// Attention over pages of keys and values (paged.hip).
#pragma once

#include "causal.hpp"

namespace ge {

// An item and the next one of its workgroup, 0 after the last. key0 is its slot, its k_lo a multiple of kPagedAlign.
struct PagedItem : CausalItem {
    uint32_t next;
};

// k and v are pools of pages, page p at p page_stride: [kv_heads][1 << page_shift rows][head_dim]. Key j of slot s
// is row j mod the page's rows of page table[s slot_pages + (j >> page_shift)].
struct PagedArgs : CausalArgs {
    const PagedItem* paged_items;  // null: in PagedInline; n_items: workgroups a KV head
    const int32_t* table;
    int64_t page_stride;
    int slot_pages, page_shift;
    // Scores x (q k unscaled) capped: cap_top tanh(cap_z x / 2 log2(e)), in log2; c is then 1. cap_top 0: as they are.
    float cap_z, cap_top;
};

// The items of a call that has few, among the kernel's arguments.
constexpr int kPagedInlineItems = 90;
struct PagedInline {
    PagedItem items[kPagedInlineItems];
};
static_assert(sizeof(PagedArgs) + sizeof(PagedInline) <= 4096, "kernel arguments");

// Rows of a wide item.
constexpr int paged_wide_rows(int hd) { return hd <= 256 ? 128 : 64; }
// Workgroups on a CU, which the registers and LDS of a launch's kernel are kept to.
constexpr int paged_workgroups(int hd) {
    return hd == 64 ? 4 : hd <= 256 ? 2 : 1;
}
constexpr int kPagedAlign = 8;  // copies are of 8 keys, which are in one page

// Head dims as causal_head_dim_ok; kinds: the CausalKind of the items.
hipError_t launch_paged(hipStream_t s, const PagedArgs& a, const PagedInline& in, int hd, bool bf16, int kinds);
// The joins' rows (splits[0] parts each; splits[1] is 0), `split` groups of lanes to a row: a power of two.
hipError_t launch_paged_join(hipStream_t s, const CausalArgs& a, const CausalInline& in, int hd, bool bf16, int split);
// Dynamic LDS limits; once per device, before launching.
hipError_t paged_configure();

}  // namespace ge
