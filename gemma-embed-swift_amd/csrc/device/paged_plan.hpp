// The plan of an attention call over pages (paged_plan.cpp).
#pragma once

#include <vector>

#include "gemmaembed.h"
#include "paged.hpp"

namespace ge {

// Workgroup w begins with items[w] and goes on along `next`.
struct PagedPlan {
    std::vector<PagedItem> items;
    std::vector<CausalJoin> joins;
    size_t workgroups = 0;  // a KV head
    size_t part_rows = 0;
    int kinds = 0, join_rows = 0, join_parts = 0;  // the most rows and parts of a join
};

// The call's sequences are checked: rows ascend, counts are under 2^30.
PagedPlan plan_paged(const ge_paged_shape& s, const ge_paged_seq* seqs, int n_seqs);

}  // namespace ge
