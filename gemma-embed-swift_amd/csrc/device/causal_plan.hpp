// The plan of a causal attention call (causal.cpp): its rows in tiles, its tiles' keys in items, and the joins of
// rows that end in more than one part.
#pragma once

#include <vector>

#include "causal.hpp"
#include "runtime_internal.hpp"

namespace ge {

constexpr int64_t kAttentionMaxRows = int64_t(1) << 30, kAttentionMaxStride = int64_t(1) << 24;

struct CausalTile {
    uint32_t base, row0, n_rows, part;
    int32_t lo, hi;  // visible keys of its rows
    uint32_t splits;
};

// Rows of one sequence, or of a run of them, against a range of their keys.
struct CausalBase {
    uint32_t q_token, key0, tile0;
    int64_t shift;
    bool direct;  // its rows have no other part
};

// What a call does, planned in a few microseconds: a call of a few dozen takes no longer on the GPU.
struct CausalPlan {
    std::vector<CausalBase> bases;
    std::vector<CausalTile> tiles;
    std::vector<uint32_t> order;  // tiles by their items' length, longest first
    std::vector<CausalJoin> joins;
    size_t n_items = 0, part_rows = 0;
    int kinds = 0, group = 1, wide = 0, key_align = 1;
};

// The plan of a call over n_seqs sequences, whose prefix of prefix_len rows is shared (0: none). An item's keys start
// at a multiple of key_align.
CausalPlan make_plan(const ge_attention_shape& s, const ge_attention_seq* seqs, int n_seqs, int64_t prefix_len, int key_align);
// The plan's items, n_items of them.
void write_items(const CausalPlan& p, CausalItem* out);

}  // namespace ge
