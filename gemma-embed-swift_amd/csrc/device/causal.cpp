// Per-op entries of causal models' attention (ge_op_attention_causal, ge_op_attention_prefix): checks,
// the plan of a call's work, and its launches.
//
// A call's rows are tiled per base: a sequence against all of its keys, the prefix's and its own, or, where
// neighbouring sequences all see the whole of a prefix that is worth it, their stacked rows against the
// prefix (read once per tile of rows and not once per sequence) and each against its own keys. Each tile's
// visible keys are split until the launch fills the GPU; rows that end in more than one part are joined by a
// second launch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <vector>

#include "causal.hpp"
#include "runtime_internal.hpp"

namespace ge {
namespace {

constexpr int kCus = 256;
constexpr int64_t kSplitMinKeys = 128;
constexpr int64_t kMaxRows = int64_t(1) << 30, kMaxStride = int64_t(1) << 24;

struct Tile {
    uint32_t base, row0, n_rows, part;
    int32_t lo, hi;  // visible keys of its rows
    uint32_t splits;
};

// Rows of one sequence, or of a run of them, against a range of their keys.
struct Base {
    uint32_t q_token, key0, tile0;
    int64_t shift;
    bool direct;  // its rows have no other part
};

// What a call does, planned in a few microseconds: a call of a few dozen takes no longer on the GPU.
struct Plan {
    std::vector<Base> bases;
    std::vector<Tile> tiles;
    std::vector<uint32_t> order;  // tiles by their items' length, longest first
    std::vector<CausalJoin> joins;
    size_t n_items = 0, part_rows = 0;
    int kinds = 0, group = 1, wide = 0;
};

int64_t divide_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
bool narrow(const Tile& t) { return t.n_rows <= uint32_t(kCausalNarrowRows); }
// 64-key steps keep the parts' blocks whole.
int32_t step_of(const Tile& t) { return t.splits > 1 ? int32_t(divide_up(t.hi - t.lo, int64_t(t.splits) * 64) * 64) : t.hi - t.lo; }

// Keys [first, end), counted through the prefix.
void add_base(Plan& p, uint32_t q_token, int64_t tokens, uint32_t key0, int64_t first, int64_t end, int64_t shift, int window,
              bool direct) {
    const uint32_t at = uint32_t(p.bases.size());
    p.bases.push_back(Base{q_token, key0, uint32_t(p.tiles.size()), shift, direct});
    const int64_t rows = tokens * p.group;
    for (int64_t r = 0; r < rows; r += p.wide) {
        const int64_t n = std::min<int64_t>(p.wide, rows - r);
        int64_t lo = first, hi = end;
        if (window) lo = std::max(first, r / p.group + shift - window + 1);
        if (shift < end) hi = std::min(end, (r + n - 1) / p.group + shift + 1);
        if (hi <= lo) lo = hi = first;
        p.tiles.push_back(Tile{at, uint32_t(r), uint32_t(n), 0, int32_t(lo), int32_t(hi), 0});
    }
}

// A wide tile's time a key on a full CU; the joining launch, with the writes and reads of its partial rows.
float wide_key_us(int head_dim) { return 0.025f * float(head_dim) / 128; }
float parts_us(int64_t rows, int kv_heads, int head_dim) { return 5.0f + float(rows) * float(kv_heads) * float(head_dim) * 8 / 3e6f; }

// Eighths of a full tile's work in the tiles of so many rows: a tile of a quarter or less is a narrow one, a
// part of a wide one spares its waves' products but not its copies.
int64_t tile_eighths(const Plan& p, int64_t rows) {
    const int64_t rest = rows % p.wide;
    return rows / p.wide * 8 + (rest == 0 ? 0 : rest <= kCausalNarrowRows ? 2 : 4 + divide_up(rest * 4, p.wide));
}

// The most keys of an item. Splitting fills the GPU and evens the items out, and costs the parts' rows
// (written, and read by the joining launch). Of no split and splits into about 1, 1.5, 2 and 3 items a CU the
// one whose estimate is least, in microseconds: a key of an item of head dim 128 takes 0.025 with one
// workgroup on a CU and 0.6 of that each with two (narrow items, which wait for memory, gain nothing by
// pairs), an item 7 besides its keys, a joining launch 5 and 1 for 3 MB of parts. Calls of short
// items (up to 128 keys) and of many even ones (four a CU unsplit, the longest no more than a CU's share of all) are
// not split. Measured, us a call unsplit / 1 / 1.5 / 2 / 3
// items a CU: one token over 20000 keys (32 heads of 128 over 8) 178 / 35 / 38 / 41 / 46, 48 tokens over 100
// to 8000 189 / 188 / 165 / 166 / 165, 128 texts over a prefix of 8192 (3 heads of 256) 332 / 200 / 178 / 215 /
// 203, one prompt of 2048 (32 heads of 128) 67 / 67 / 78 / 83 / 84. A token over 32768 keys beside 127 over
// 100: 293 unsplit, 54 split.
int64_t split_limit(const Plan& p, int kv_heads, int head_dim) {
    constexpr int kBins = 64;
    const float key_us = wide_key_us(head_dim);
    int64_t total = 0, longest = 0, wide_keys = 0;
    for (const Tile& t : p.tiles) {
        const int64_t n = t.hi - t.lo;
        total += n;
        wide_keys += narrow(t) ? 0 : n;
        longest = std::max(longest, n);
    }
    const float pair = 2 * wide_keys >= total ? 0.6f : 1.0f;
    if (longest <= kSplitMinKeys ||
        (int64_t(p.tiles.size()) * kv_heads >= 4 * kCus && float(longest) <= float(total * kv_heads) * pair / kCus))
        return std::max<int64_t>(longest, 64);
    int64_t best = longest;
    float best_us = 1e30f;
    for (const float per_cu : {0.0f, 1.0f, 1.5f, 2.0f, 3.0f}) {
        const int64_t limit =
            per_cu == 0.0f ? longest : std::max(kSplitMinKeys, (int64_t(float(total * kv_heads) / (per_cu * kCus)) + 63) / 64 * 64);
        if (per_cu != 0.0f && limit >= longest) continue;
        // items by their keys, in kBins steps
        int count[kBins] = {}, items = 0;
        int64_t parts = 0;
        const float inv = 1.0f / float(limit), to_bin = kBins / float(limit + 1);
        for (const Tile& t : p.tiles) {
            const int n = t.hi - t.lo;
            if (!n) continue;
            const int k = n <= limit ? 1 : int(std::ceil(float(n) * inv));
            count[std::min(kBins - 1, int(float(n) / float(k) * to_bin))] += k * kv_heads;
            items += k * kv_heads;
            if (k > 1 || !p.bases[t.base].direct) parts += int64_t(k) * t.n_rows;
        }
        // at least the work at the rate of full CUs, and, with the items started longest first, two a CU, the
        // end of the first of each round's first and second half
        float us = float(total) * float(kv_heads) * key_us * pair / kCus;
        int k = 0, seen = 0;
        for (int bin = kBins - 1; bin >= 0; bin--) {
            seen += count[bin];
            for (; k < seen; k += kCus)
                us = std::max(us, (float(k / (2 * kCus)) * 2 * pair + (k / kCus % 2 ? 2 * pair : 1.0f)) * key_us * float(limit) * float(bin + 1) / kBins);
        }
        us += 7.0f * float((items + 2 * kCus - 1) / (2 * kCus));
        if (parts) us += parts_us(parts, kv_heads, head_dim);
        if (us < best_us) {
            best_us = us;
            best = limit;
        }
    }
    return best;
}

Plan make_plan(const ge_attention_shape& s, const ge_attention_seq* seqs, int n_seqs, int64_t prefix_len) {
    Plan p;
    p.group = s.heads / s.kv_heads;
    p.wide = causal_wide_rows(s.head_dim);
    p.bases.reserve(size_t(n_seqs) * (prefix_len ? 2 : 1));
    p.tiles.reserve(size_t(n_seqs) * 2 + 64);
    struct Use {
        int own = -1, prefix = -1;
        int64_t prefix_row = 0;  // the sequence's first row in its prefix base
    };
    std::vector<Use> use(size_t(n_seqs), Use{});
    // Sequences whose every row sees the whole prefix, wherever it stands, may stack up.
    auto stacks = [&](const ge_attention_seq& q) { return prefix_len && s.window == 0 && int64_t(q.q_len) <= int64_t(q.kv_len) + 1; };
    for (int i = 0; i < n_seqs;) {
        if (!seqs[i].q_len) {
            i++;
            continue;
        }
        const uint32_t q_start = seqs[i].q_start;
        int64_t tokens = 0, apart = 0;  // of the run from i to j
        bool alone = true;
        int j = i;
        do {
            tokens += seqs[j].q_len;
            apart += tile_eighths(p, int64_t(seqs[j].q_len) * p.group);
            alone = alone && seqs[j].kv_len == 0;
            j++;
        } while (stacks(seqs[j - 1]) && j < n_seqs && seqs[j].q_len && stacks(seqs[j]) && seqs[j].q_start == q_start + uint64_t(tokens));
        // Stacked, the run has fewer tiles to take over the prefix, but two parts a row to join. Of n sequences,
        // us apart / stacked over 24, 400, 1000 and 4000 keys: one token of 4 heads over each of 2 KV heads of 128,
        // n = 256: 25 / 36, 31 / 40, 38 / 40, 74 / 45; 4 to 32 tokens of 3 heads of 256, n = 96: 25 / 35, 42 / 44,
        // 53 / 48, 91 / 69; 20 to 100 tokens of 4 heads over each of 8 of 64, n = 256: 67 / 214, 126 / 246,
        // 227 / 326, 641 / 698.
        const int64_t rows = tokens * p.group;
        const bool stack = j > i + 1 && float(apart - tile_eighths(p, rows)) / 8 * float(prefix_len) * float(s.kv_heads) *
                                                wide_key_us(s.head_dim) / kCus > (alone ? 0.0f : parts_us(2 * rows, s.kv_heads, s.head_dim));
        int64_t row = 0;
        if (stack) add_base(p, q_start, tokens, 0, 0, prefix_len, kMaxRows, 0, alone);
        const int prefix = int(p.bases.size()) - 1;
        for (; i < j; i++) {
            const ge_attention_seq& e = seqs[i];
            if (stack) {
                use[size_t(i)].prefix = prefix;
                use[size_t(i)].prefix_row = row;
                row += int64_t(e.q_len) * p.group;
                if (!e.kv_len) continue;
            }
            use[size_t(i)].own = int(p.bases.size());
            add_base(p, e.q_start, e.q_len, e.kv_start, stack ? prefix_len : 0, prefix_len + e.kv_len,
                     prefix_len + e.kv_len - int64_t(e.q_len), s.window, !stack);
        }
    }

    const int64_t limit = split_limit(p, s.kv_heads, s.head_dim);
    // The longest items first, so that the last ones to start are short: tiles by their items' keys (a wide
    // item's weighing four times), in 256 steps.
    constexpr int kSteps = 256;
    const int64_t heaviest = 4 * std::max<int64_t>(limit, 1);
    auto place = [&](const Tile& t) { return kSteps - 1 - int(int64_t(step_of(t)) * (narrow(t) ? 1 : 4) * (kSteps - 1) / heaviest); };
    uint32_t first[kSteps + 1] = {};
    bool joined = false;
    for (Tile& t : p.tiles) {
        const bool direct = p.bases[t.base].direct;
        t.splits = uint32_t(divide_up(t.hi - t.lo, limit));
        t.part = uint32_t(p.part_rows);
        if (direct && t.splits <= 1) {
            t.splits = 1;  // also where its rows see nothing: they are written
        } else {
            joined = true;
            p.part_rows += size_t(t.splits) * t.n_rows;
            if (p.part_rows >= kDirect) fail(GE_ERR_INVALID, "attention: the call's rows and keys are too many for one call");
        }
        p.n_items += t.splits;
        if (t.splits) p.kinds |= narrow(t) ? kCausalNarrow : kCausalWide;
        first[place(t) + 1]++;
    }
    for (int i = 0; i < kSteps; i++) first[i + 1] += first[i];
    p.order.resize(p.tiles.size());
    for (size_t i = 0; i < p.tiles.size(); i++) p.order[first[place(p.tiles[i])]++] = uint32_t(i);

    if (joined) p.joins.reserve(size_t(n_seqs) + p.tiles.size());
    for (int i = 0; joined && i < n_seqs; i++) {
        const Use& u = use[size_t(i)];
        const Base* const side[2] = {u.own >= 0 ? &p.bases[size_t(u.own)] : nullptr, u.prefix >= 0 ? &p.bases[size_t(u.prefix)] : nullptr};
        const int64_t start[2] = {0, u.prefix_row}, rows = int64_t(seqs[i].q_len) * p.group;
        for (int64_t r = 0; r < rows;) {
            CausalJoin j{seqs[i].q_start, uint32_t(r), 0, {}, {}, {}};
            int64_t end = rows;
            bool written = false;
            for (int k = 0; k < 2; k++) {
                if (!side[k]) continue;
                const int64_t at = start[k] + r;
                const Tile& t = p.tiles[side[k]->tile0 + size_t(at / p.wide)];
                j.part[k] = t.part + uint32_t(at - t.row0);
                j.stride[k] = t.n_rows;
                j.splits[k] = t.splits;
                end = std::min(end, int64_t(t.row0) + t.n_rows - start[k]);
                written = written || (side[k]->direct && t.splits == 1);
            }
            j.n_rows = uint32_t(end - r);
            if (!written) p.joins.push_back(j);
            r = end;
        }
    }
    return p;
}

// The plan's items, n_items of them.
void write_items(const Plan& p, CausalItem* out) {
    for (const uint32_t i : p.order) {
        const Tile& t = p.tiles[i];
        const Base& b = p.bases[t.base];
        const int32_t step = step_of(t);
        for (uint32_t s = 0; s < t.splits; s++) {
            const int32_t k = t.lo + int32_t(s) * step;
            const bool direct = b.direct && t.splits == 1;
            *out++ = CausalItem{b.q_token, t.row0, t.n_rows, b.key0, uint32_t(std::min(k, t.hi)), uint32_t(std::min(k + step, t.hi)),
                                int32_t(b.shift), direct ? kDirect : t.part + s * t.n_rows, narrow(t)};
        }
    }
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

void check_stride(const char* what, int64_t& stride, int64_t width) {
    if (stride == 0) stride = width;
    if (stride < width || stride % 8 || stride > kMaxStride)
        fail(GE_ERR_INVALID, "attention: %s row stride %lld (a multiple of 8 from %lld to %lld elements, or 0)", what,
             static_cast<long long>(stride), static_cast<long long>(width), static_cast<long long>(kMaxStride));
}

void attend(ge_ctx* c, const ge_attention_shape* shape, const void* q, const void* prefix_k, const void* prefix_v,
            int64_t prefix_len, const void* k, const void* v, const ge_attention_seq* seqs, int n_seqs, void* out) {
    if (!shape) fail(GE_ERR_INVALID, "attention: null shape");
    ge_attention_shape s = *shape;
    if (s.type != GE_TYPE_F16 && s.type != GE_TYPE_BF16) fail(GE_ERR_INVALID, "attention: type %d is neither F16 nor BF16", s.type);
    if (!causal_head_dim_ok(s.head_dim)) fail(GE_ERR_INVALID, "attention: head dim %d (64, 128, 256 or 512)", s.head_dim);
    if (s.heads <= 0 || s.kv_heads <= 0 || s.heads % s.kv_heads || s.heads > 4096)
        fail(GE_ERR_INVALID, "attention: %d query heads over %d KV heads (a multiple, up to 4096)", s.heads, s.kv_heads);
    if (s.q_rows < 0 || s.kv_rows < 0 || prefix_len < 0 || s.q_rows >= kMaxRows || s.kv_rows >= kMaxRows ||
        int64_t(s.kv_rows) + prefix_len >= kMaxRows || s.window < 0 || s.window >= kMaxRows || n_seqs < 0)
        fail(GE_ERR_INVALID, "attention: query rows, window, sequences, and key rows and prefix together from 0 to under 2^30");
    if (int64_t(s.q_rows) * (s.heads / s.kv_heads) >= kMaxRows)
        fail(GE_ERR_INVALID, "attention: %d rows of %d query heads a KV head pass 2^30", s.q_rows, s.heads / s.kv_heads);
    if (!std::isfinite(s.scale)) fail(GE_ERR_INVALID, "attention: scale is not finite");
    const int64_t kv_width = int64_t(s.kv_heads) * s.head_dim, q_width = int64_t(s.heads) * s.head_dim;
    check_stride("q", s.q_stride, q_width);
    check_stride("k", s.k_stride, kv_width);
    check_stride("v", s.v_stride, kv_width);
    check_stride("out", s.out_stride, q_width);
    if (n_seqs == 0) return;
    if (!seqs) fail(GE_ERR_INVALID, "attention: null sequences");
    uint64_t q_end = 0, kv_end = 0;
    for (int i = 0; i < n_seqs; i++) {
        const ge_attention_seq& e = seqs[i];
        if (e.q_start < q_end && e.q_len) fail(GE_ERR_INVALID, "attention: sequence %d's query rows start before the last one's end", i);
        if (uint64_t(e.q_start) + e.q_len > uint64_t(s.q_rows) || uint64_t(e.kv_start) + e.kv_len > uint64_t(s.kv_rows))
            fail(GE_ERR_INVALID, "attention: sequence %d: query rows [%u, +%u) of %d, key rows [%u, +%u) of %d", i, e.q_start,
                 e.q_len, s.q_rows, e.kv_start, e.kv_len, s.kv_rows);
        if (e.q_len) q_end = uint64_t(e.q_start) + e.q_len;
        if (e.q_len && e.kv_len) kv_end = 1;
    }
    if (q_end == 0) return;
    if (!q || !out || (kv_end && (!k || !v)) || (prefix_len && (!prefix_k || !prefix_v)))
        fail(GE_ERR_INVALID, "attention: q, out, and k and v of every key row");
    if (!aligned(q) || !aligned(k) || !aligned(v) || !aligned(out) || !aligned(prefix_k) || !aligned(prefix_v))
        fail(GE_ERR_INVALID, "attention: buffers are 16-byte aligned");

    if (!c->causal_ready) {
        hip_check(causal_configure(), "hipFuncSetAttribute");
        c->causal_ready = true;
    }
    const Plan p = make_plan(s, seqs, n_seqs, prefix_len);
    if (p.n_items * uint64_t(s.kv_heads) > kCausalMaxGroups || p.joins.size() * uint64_t(s.kv_heads) > kCausalMaxGroups)
        fail(GE_ERR_INVALID, "attention: the call's rows and keys are too many for one call");
    OpTemps temps(c);
    CausalInline in;
    const bool few = p.n_items <= size_t(kCausalInlineItems) && p.joins.size() <= size_t(kCausalInlineJoins);
    const size_t item_bytes = (p.n_items * sizeof(CausalItem) + 255) / 256 * 256;
    unsigned char* const lists = few ? nullptr : op_lists(c, item_bytes + p.joins.size() * sizeof(CausalJoin));
    write_items(p, few ? in.items : reinterpret_cast<CausalItem*>(lists));
    std::copy(p.joins.begin(), p.joins.end(), few ? in.joins : reinterpret_cast<CausalJoin*>(lists + item_bytes));
    const size_t o_at = temps.reserve(p.part_rows * size_t(kv_width) * 4);
    const size_t ml_at = temps.reserve(p.part_rows * size_t(s.kv_heads) * 8);
    unsigned char* const base = p.part_rows ? temps.base() : nullptr;

    CausalArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k);
    a.v = static_cast<const uint16_t*>(v);
    a.prefix_k = static_cast<const uint16_t*>(prefix_k);
    a.prefix_v = static_cast<const uint16_t*>(prefix_v);
    a.out = static_cast<uint16_t*>(out);
    a.items = reinterpret_cast<const CausalItem*>(lists);
    a.joins = few ? nullptr : reinterpret_cast<const CausalJoin*>(lists + item_bytes);
    a.part_o = reinterpret_cast<float*>(base + o_at);
    a.part_ml = reinterpret_cast<float2*>(base + ml_at);
    a.q_stride = s.q_stride;
    a.k_stride = s.k_stride;
    a.v_stride = s.v_stride;
    a.out_stride = s.out_stride;
    a.part_rows = p.part_rows;
    a.n_items = int(p.n_items);
    a.n_joins = int(p.joins.size());
    for (const CausalJoin& j : p.joins) a.join_rows = std::max(a.join_rows, int(j.n_rows));
    a.prefix_len = int(prefix_len);
    a.group = s.heads / s.kv_heads;
    a.kv_heads = s.kv_heads;
    a.window = s.window;
    // a hidden key's -inf times this stays -inf, also at scale 0
    a.c = std::min(std::max(std::fabs(s.scale) * 1.4426950408889634f, FLT_MIN), FLT_MAX);
    a.q_flip = s.scale < 0.0f ? 0x80008000u : 0u;
    launch(c, "attention_causal", [&] { return launch_causal(c->stream, a, in, s.head_dim, s.type == GE_TYPE_BF16, p.kinds); });
    if (a.n_joins)
        launch(c, "attention_join", [&] { return launch_causal_join(c->stream, a, in, s.head_dim, s.type == GE_TYPE_BF16); });
    hip_check(hipStreamSynchronize(c->stream), "hipStreamSynchronize");
}

}  // namespace
}  // namespace ge

extern "C" {

int ge_op_attention_causal(ge_ctx* c, const ge_attention_shape* shape, const void* q, const void* k, const void* v,
                           const ge_attention_seq* seqs, int32_t n_seqs, void* out) {
    return ge::guarded(c, [&] { ge::attend(c, shape, q, nullptr, nullptr, 0, k, v, seqs, n_seqs, out); });
}

int ge_op_attention_prefix(ge_ctx* c, const ge_attention_shape* shape, const void* q, const void* prefix_k,
                           const void* prefix_v, int32_t prefix_len, const void* k, const void* v,
                           const ge_attention_seq* seqs, int32_t n_seqs, void* out) {
    return ge::guarded(c, [&] { ge::attend(c, shape, q, prefix_k, prefix_v, prefix_len, k, v, seqs, n_seqs, out); });
}

}  // extern "C"
