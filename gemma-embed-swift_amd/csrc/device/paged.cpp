// Per-op entries of a paged cache: rotary positions (ge_op_rotary_create, ge_op_rotate_heads), page tables
// (ge_op_page_table_create, ge_op_page_table_set), appending (ge_op_paged_append) and attention
// (ge_op_attention_paged).
//
// A page table is kept twice: on the device for the kernels and on the host, where every call's sequences are
// checked against it, so that a kernel never meets a page that is not there.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <memory>
#include <vector>

#include "paged_plan.hpp"
#include "rotary.hpp"
#include "runtime_internal.hpp"

struct ge_rotary {
    ge_ctx* ctx = nullptr;
    int dims = 0, layout = 0;
    float fade = 1.0f, gain = 1.0f;
    double* turns = nullptr;
};

struct ge_page_table {
    ge_ctx* ctx = nullptr;
    int slots = 0, slot_pages = 0, page_rows = 0, page_shift = 0, n_pages = 0;
    std::vector<int32_t> pages;  // [slots][slot_pages], -1 where there is none
    // Each slot's last run of pages with none missing: [begin, end).
    struct Run {
        int begin, end;
    };
    std::vector<Run> runs;
    // The sequence of the last append that wrote each page, counted through the calls: up to the highest page set.
    mutable std::vector<uint32_t> writer;
    mutable uint32_t writers = 0;
    int32_t* dev = nullptr;
};

namespace ge {
namespace {

constexpr double kTwoPi = 6.283185307179586476925286766559;
constexpr int64_t kAttentionMaxRows = int64_t(1) << 30, kAttentionMaxStride = int64_t(1) << 24;
constexpr int64_t kMaxTable = int64_t(1) << 28, kMaxPages = int64_t(1) << 28;
constexpr int kMaxHeads = 4096, kMaxPageRows = 1024;
constexpr float kMaxCap = 1024.0f;  // for its accuracy (Capped, paged.hip)

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

void check_rows_stride(const char* op, const char* what, int64_t& stride, int64_t width, int multiple) {
    if (stride == 0) stride = width;
    if (stride < width || stride % multiple || stride > kAttentionMaxStride)
        fail(GE_ERR_INVALID, "%s: %s row stride %lld (a multiple of %d from %lld to %lld elements, or 0)", op, what,
             static_cast<long long>(stride), multiple, static_cast<long long>(width), static_cast<long long>(kAttentionMaxStride));
}

// Elements of a page, of kv_heads heads.
int64_t page_elements(const ge_page_table* t, int kv_heads, int head_dim) {
    return int64_t(t->page_rows) * kv_heads * head_dim;
}

void check_page_stride(const char* op, int64_t& stride, int64_t elements) {
    if (stride == 0) stride = elements;
    if (stride < elements || stride % 8 || stride > (int64_t(1) << 40))
        fail(GE_ERR_INVALID, "%s: page stride %lld (a multiple of 8 from %lld elements on, or 0)", op, static_cast<long long>(stride),
             static_cast<long long>(elements));
}

// Whether the slot has all of its pages [begin, end).
bool has_pages(const ge_page_table* t, uint32_t slot, int64_t begin, int64_t end) {
    const ge_page_table::Run& r = t->runs[slot];
    if (begin >= end || (r.begin <= begin && end <= r.end)) return true;
    const int32_t* const p = t->pages.data() + size_t(slot) * size_t(t->slot_pages);
    return std::all_of(p + begin, p + end, [](int32_t page) { return page >= 0; });
}

// Rows and slots of a call's sequences; returns the end of the last one's rows.
int64_t check_seqs(const char* op, const ge_page_table* t, const ge_paged_seq* seqs, int n_seqs, int rows) {
    uint64_t end = 0;
    for (int i = 0; i < n_seqs; i++) {
        const ge_paged_seq& e = seqs[i];
        if (e.q_start < end && e.q_len) fail(GE_ERR_INVALID, "%s: sequence %d's query rows start before the last one's end", op, i);
        if (uint64_t(e.q_start) + e.q_len > uint64_t(rows))
            fail(GE_ERR_INVALID, "%s: sequence %d: query rows [%u, +%u) of %d", op, i, e.q_start, e.q_len, rows);
        if (e.slot >= uint32_t(t->slots)) fail(GE_ERR_INVALID, "%s: sequence %d: slot %u of %d", op, i, e.slot, t->slots);
        if (e.kv_len > uint64_t(t->slot_pages) * uint64_t(t->page_rows))
            fail(GE_ERR_INVALID, "%s: sequence %d: %u keys in %d pages of %d rows", op, i, e.kv_len, t->slot_pages, t->page_rows);
        if (e.q_len) end = uint64_t(e.q_start) + e.q_len;
    }
    return int64_t(end);
}

void check_table(const char* op, const ge_ctx* c, const ge_page_table* t) {
    if (!t) fail(GE_ERR_INVALID, "%s: null page table", op);
    if (t->ctx != c) fail(GE_ERR_INVALID, "%s: the page table is another context's", op);
}

// ---------------------------------------------------------------------------- rotary positions

std::vector<double> rotary_turns(const ge_rotary_desc& d) {
    std::vector<double> turns(size_t(d.dims) / 2);
    for (size_t i = 0; i < turns.size(); i++) {
        double t = std::pow(double(d.base), -2.0 * double(i) / d.dims) / kTwoPi;
        if (d.scaling == GE_ROTARY_LINEAR) t /= d.factor;
        if (d.scaling == GE_ROTARY_BY_TURNS) {
            const double low = d.low_turns, high = d.high_turns;
            const double w = std::min(std::max((d.trained * t - low) / (high - low), 0.0), 1.0);
            t *= w + (1.0 - w) / d.factor;
        }
        turns[i] = t;
    }
    return turns;
}

void check_rotary(const ge_rotary_desc& d) {
    if (d.dims <= 0 || d.dims % 2 || d.dims > 512) fail(GE_ERR_INVALID, "rotary: %d elements (an even number from 2 to 512)", d.dims);
    if (d.layout != GE_ROTARY_HALVES && d.layout != GE_ROTARY_PAIRS) fail(GE_ERR_INVALID, "rotary: layout %d", d.layout);
    if (d.scaling < GE_ROTARY_PLAIN || d.scaling > GE_ROTARY_BY_TURNS) fail(GE_ERR_INVALID, "rotary: scaling %d", d.scaling);
    if (!(d.base > 0.0f) || !std::isfinite(d.base)) fail(GE_ERR_INVALID, "rotary: base must be positive and finite");
    if (!std::isfinite(d.magnitude)) fail(GE_ERR_INVALID, "rotary: magnitude is not finite");
    // (sines and cosines times it are fp32 values)
    if (d.magnitude != 0.0f && std::fabs(d.magnitude) < FLT_MIN) fail(GE_ERR_INVALID, "rotary: magnitude below 2^-126 and not 0");
    if (d.scaling != GE_ROTARY_PLAIN && (!(d.factor > 0.0f) || !std::isfinite(d.factor)))
        fail(GE_ERR_INVALID, "rotary: factor must be positive and finite");
    if (d.scaling == GE_ROTARY_BY_TURNS &&
        (d.trained <= 0 || !std::isfinite(d.low_turns) || !std::isfinite(d.high_turns) || !(d.low_turns < d.high_turns)))
        fail(GE_ERR_INVALID, "rotary: by turns needs trained > 0 and low_turns < high_turns");
}

// ---------------------------------------------------------------------------- rows of heads

constexpr const char* kRotate = "rotate_heads";
constexpr const char* kAppend = "paged_append";

// The checks and arguments of both entries over rows of heads.
HeadsArgs heads_args(const char* op, ge_ctx* c, const ge_heads_shape* shape, const ge_rotary* r, bool append, ge_heads_shape* checked) {
    if (!shape) fail(GE_ERR_INVALID, "%s: null shape", op);
    ge_heads_shape s = *shape;
    if (s.type != GE_TYPE_F16 && s.type != GE_TYPE_BF16) fail(GE_ERR_INVALID, "%s: results of type %d (F16 or BF16)", op, s.type);
    if (s.in_type != GE_TYPE_F32 && s.in_type != s.type) fail(GE_ERR_INVALID, "%s: inputs of type %d (F32, or the results')", op, s.in_type);
    if (s.heads < 0 || s.kv_heads < 0 || s.heads > kMaxHeads || s.kv_heads > kMaxHeads || s.heads + s.kv_heads == 0)
        fail(GE_ERR_INVALID, "%s: %d query and %d KV heads (0 to %d, not both 0)", op, s.heads, s.kv_heads, kMaxHeads);
    if (s.head_dim <= 0 || s.head_dim % 2 || s.head_dim > 512)
        fail(GE_ERR_INVALID, "%s: head dim %d (an even number from 2 to 512)", op, s.head_dim);
    if (s.rows < 0 || s.rows >= kAttentionMaxRows) fail(GE_ERR_INVALID, "%s: %d rows (0 to under 2^30)", op, s.rows);
    if (s.normed & ~(append ? GE_NORM_Q | GE_NORM_K | GE_NORM_V : GE_NORM_Q | GE_NORM_K))
        fail(GE_ERR_INVALID, "%s: norms %d", op, s.normed);
    if (s.normed && !(s.eps >= 0.0f && std::isfinite(s.eps))) fail(GE_ERR_INVALID, "%s: eps must be finite and not negative", op);
    if (r && r->ctx != c) fail(GE_ERR_INVALID, "%s: the rotary positions are another context's", op);
    if (r && r->dims > s.head_dim) fail(GE_ERR_INVALID, "%s: %d elements to turn in a head of %d", op, r->dims, s.head_dim);
    const int64_t q_width = int64_t(s.heads) * s.head_dim, kv_width = int64_t(s.kv_heads) * s.head_dim;
    check_rows_stride(op, "q", s.q_stride, q_width, 1);
    check_rows_stride(op, "k", s.k_stride, kv_width, 1);
    check_rows_stride(op, "q_out", s.q_out_stride, q_width, 1);
    if (append)
        check_rows_stride(op, "v", s.v_stride, kv_width, 1);
    else
        check_rows_stride(op, "k_out", s.k_out_stride, kv_width, 1);

    HeadsArgs a{};
    a.q_stride = s.q_stride;
    a.k_stride = s.k_stride;
    a.v_stride = s.v_stride;
    a.q_out_stride = s.q_out_stride;
    a.k_out_stride = s.k_out_stride;
    a.heads = s.heads;
    a.kv_heads = s.kv_heads;
    a.head_dim = s.head_dim;
    a.rows = s.rows;
    a.normed = s.normed;
    a.eps = s.eps;
    a.fade = a.gain = 1.0f;
    if (r) {
        a.turns = r->turns;
        a.half = r->dims / 2;
        a.pairs = r->layout == GE_ROTARY_PAIRS;
        a.fade = r->fade;
        a.gain = r->gain;
    }
    *checked = s;
    return a;
}

// Operands by their part: null where there are none of its heads.
struct Operand {
    const char* name;
    const void* p;
    bool needed;
    int size;   // of an element
    bool rows;  // read or written a unit at a time
};

// Checks them and returns the unit of a call: the largest that its heads, the part that turns, its strides and its
// addresses come in together, accesses being of 16 bytes at most. (One rule: a unit that one of them refuses may leave
// only a smaller one than the next, as heads past 256 elements do, which come in units of 4 and 1 but not of 2.)
int operands_unit(const char* op, const ge_heads_shape& s, int half, bool append, std::initializer_list<Operand> list) {
    for (const Operand& o : list) {
        if (o.needed && !o.p) fail(GE_ERR_INVALID, "%s: null %s", op, o.name);
        if (!aligned(o.p, size_t(o.size))) fail(GE_ERR_INVALID, "%s: %s is not aligned to its elements", op, o.name);
    }
    const auto moves_in = [&](int u) {
        const int in = std::min(u, s.in_type == GE_TYPE_F32 ? 4 : 8);
        return heads_unit_ok(s.head_dim, half, u) && s.q_stride % in == 0 && s.k_stride % in == 0 && s.q_out_stride % u == 0 &&
               (append ? s.v_stride % in == 0 : s.k_out_stride % u == 0) &&
               std::all_of(list.begin(), list.end(), [&](const Operand& o) { return !o.rows || aligned(o.p, size_t(std::min(16, u * o.size))); });
    };
    int unit = 8;
    while (!moves_in(unit)) unit /= 2;  // in units of 1 it does
    return unit;
}

// Results may take their operand's place row by row and head by head, where both are of one type.
void check_in_place(const char* op, const char* what, const ge_heads_shape& s, const void* in, int64_t in_stride, const void* out,
                    int64_t out_stride) {
    if (in && in == out && (s.in_type != s.type || (s.rows > 1 && in_stride != out_stride)))
        fail(GE_ERR_INVALID, "%s: %s in its own place, of another type or row stride", op, what);
}

void rotate(ge_ctx* c, const ge_heads_shape* shape, const ge_rotary* r, const void* q, const void* k, const void* q_norm,
            const void* k_norm, const void* positions, void* q_out, void* k_out) {
    ge_heads_shape s;
    HeadsArgs a = heads_args(kRotate, c, shape, r, false, &s);
    if (s.rows == 0) return;
    const int in = s.in_type == GE_TYPE_F32 ? 4 : 2;
    const int unit = operands_unit(kRotate, s, a.half, false,
                                   {{"q", q, s.heads > 0, in, true}, {"k", k, s.kv_heads > 0, in, true}, {"q_out", q_out, s.heads > 0, 2, true},
                                    {"k_out", k_out, s.kv_heads > 0, 2, true}, {"q_norm", q_norm, false, 4, false}, {"k_norm", k_norm, false, 4, false}});
    check_in_place(kRotate, "q", s, q, s.q_stride, q_out, s.q_out_stride);
    check_in_place(kRotate, "k", s, k, s.k_stride, k_out, s.k_out_stride);
    if (r && !positions) fail(GE_ERR_INVALID, "%s: null positions", kRotate);
    if (!aligned(positions, 4)) fail(GE_ERR_INVALID, "%s: positions are not aligned to their elements", kRotate);
    a.q = q;
    a.k = k;
    a.q_out = static_cast<uint16_t*>(q_out);
    a.k_out = static_cast<uint16_t*>(k_out);
    a.q_norm = static_cast<const float*>(q_norm);
    a.k_norm = static_cast<const float*>(k_norm);
    a.positions = static_cast<const int32_t*>(positions);
    a.rows_each = heads_rows_each(s.rows);
    launch(c, kRotate, [&] { return launch_rotate_heads(c->stream, a, s.in_type == GE_TYPE_F32, s.type == GE_TYPE_BF16, unit); });
    hip_check(hipStreamSynchronize(c->stream), "hipStreamSynchronize");
}

// Notes the pages that a call's sequences write; a page is written by one sequence of a call, at one place of its
// slot.
void claim_pages(const ge_page_table* t, const ge_paged_seq* seqs, int n_seqs) {
    if (t->writers > 0xffffffffu - uint32_t(n_seqs) - 1) {
        std::fill(t->writer.begin(), t->writer.end(), 0u);
        t->writers = 0;
    }
    const uint32_t first = t->writers + 1;
    t->writers += uint32_t(n_seqs);
    for (int i = 0; i < n_seqs; i++) {
        const ge_paged_seq& e = seqs[i];
        if (!e.q_len) continue;
        const int32_t* const pages = t->pages.data() + size_t(e.slot) * size_t(t->slot_pages);
        for (uint32_t j = (e.kv_len - e.q_len) >> t->page_shift; j <= (e.kv_len - 1) >> t->page_shift; j++) {
            uint32_t& w = t->writer[size_t(pages[j])];
            if (w >= first) fail(GE_ERR_INVALID, "%s: page %d is written by sequence %u and again by sequence %d", kAppend, pages[j], w - first, i);
            w = first + uint32_t(i);
        }
    }
}

void append(ge_ctx* c, const ge_heads_shape* shape, const ge_rotary* r, const void* q, const void* k, const void* v,
            const void* q_norm, const void* k_norm, const void* positions, const ge_page_table* t, const ge_paged_seq* seqs,
            int n_seqs, void* q_out, void* k_pages, void* v_pages) {
    ge_heads_shape s;
    HeadsArgs a = heads_args(kAppend, c, shape, r, true, &s);
    check_table(kAppend, c, t);
    if (s.kv_heads == 0) fail(GE_ERR_INVALID, "%s: no KV heads", kAppend);
    if (n_seqs < 0) fail(GE_ERR_INVALID, "%s: %d sequences", kAppend, n_seqs);
    check_page_stride(kAppend, s.page_stride, page_elements(t, s.kv_heads, s.head_dim));
    if (n_seqs == 0) return;
    if (!seqs) fail(GE_ERR_INVALID, "%s: null sequences", kAppend);
    if (check_seqs(kAppend, t, seqs, n_seqs, s.rows) == 0) return;
    int64_t rows = 0;
    for (int i = 0; i < n_seqs; i++) {
        const ge_paged_seq& e = seqs[i];
        if (!e.q_len) continue;
        if (e.q_len > e.kv_len) fail(GE_ERR_INVALID, "%s: sequence %d: %u new keys of %u", kAppend, i, e.q_len, e.kv_len);
        if (!has_pages(t, e.slot, (e.kv_len - e.q_len) >> t->page_shift, int64_t((e.kv_len - 1) >> t->page_shift) + 1))
            fail(GE_ERR_INVALID, "%s: sequence %d: slot %u lacks a page of keys [%u, %u)", kAppend, i, e.slot, e.kv_len - e.q_len, e.kv_len);
        rows += e.q_len;
    }
    const int in = s.in_type == GE_TYPE_F32 ? 4 : 2;
    const int unit = operands_unit(kAppend, s, a.half, true,
                                   {{"q", q, s.heads > 0, in, true}, {"k", k, true, in, true}, {"v", v, true, in, true}, {"q_out", q_out, s.heads > 0, 2, true},
                                    {"k_pages", k_pages, true, 2, true}, {"v_pages", v_pages, true, 2, true}, {"q_norm", q_norm, false, 4, false},
                                    {"k_norm", k_norm, false, 4, false}});
    check_in_place(kAppend, "q", s, q, s.q_stride, q_out, s.q_out_stride);
    if (!aligned(positions, 4)) fail(GE_ERR_INVALID, "%s: positions are not aligned to their elements", kAppend);
    claim_pages(t, seqs, n_seqs);

    // few sequences: one item each; many: one for each workgroup, which need not search them then
    const uint32_t each = uint32_t(heads_rows_each(int(rows)));
    size_t groups = 0, some = 0;
    for (int i = 0; i < n_seqs; i++) {
        groups += (size_t(seqs[i].q_len) + each - 1) / each;
        some += seqs[i].q_len > 0;
    }
    if (groups > kCausalMaxGroups) fail(GE_ERR_INVALID, "%s: %zu sequences with rows are too many for one call", kAppend, some);
    const bool inlined = some <= size_t(kAppendInlineItems);
    OpTemps temps(c);
    AppendInline few;
    AppendItem* const list = inlined ? few.items : reinterpret_cast<AppendItem*>(op_lists(c, groups * sizeof(AppendItem)));
    AppendItem* out = list;
    uint32_t group = 0;
    for (int i = 0; i < n_seqs; i++) {
        const ge_paged_seq& e = seqs[i];
        const uint32_t piece = inlined ? e.q_len : each;
        for (uint32_t at = 0; at < e.q_len; at += piece) {
            const uint32_t n = std::min(piece, e.q_len - at);
            *out++ = AppendItem{e.q_start + at, n, e.slot, e.kv_len - e.q_len + at, group};
            group += (n + each - 1) / each;
        }
    }
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_out = static_cast<uint16_t*>(q_out);
    a.k_out = static_cast<uint16_t*>(k_pages);
    a.v_out = static_cast<uint16_t*>(v_pages);
    a.q_norm = static_cast<const float*>(q_norm);
    a.k_norm = static_cast<const float*>(k_norm);
    a.positions = static_cast<const int32_t*>(positions);
    a.table = t->dev;
    a.items = inlined ? nullptr : list;
    a.n_items = int(out - list);
    a.workgroups = int(groups);
    a.rows_each = int(each);
    a.slot_pages = t->slot_pages;
    a.page_shift = t->page_shift;
    a.page_stride = s.page_stride;
    launch(c, kAppend, [&] { return launch_append(c->stream, a, few, s.in_type == GE_TYPE_F32, s.type == GE_TYPE_BF16, unit); });
    hip_check(hipStreamSynchronize(c->stream), "hipStreamSynchronize");
}

// ---------------------------------------------------------------------------- page tables

// A slot's run, from its pages.
ge_page_table::Run find_run(const ge_page_table* t, uint32_t slot) {
    const int32_t* const p = t->pages.data() + size_t(slot) * size_t(t->slot_pages);
    int end = t->slot_pages;
    while (end > 0 && p[end - 1] < 0) end--;
    int begin = end;
    while (begin > 0 && p[begin - 1] >= 0) begin--;
    return {begin, end};
}

void set_pages(ge_ctx* c, ge_page_table* t, const ge_page_entry* entries, int n) {
    check_table("page_table_set", c, t);
    if (n < 0 || (n > 0 && !entries)) fail(GE_ERR_INVALID, "page_table_set: null entries");
    int32_t highest = -1;
    for (int i = 0; i < n; i++) {
        const ge_page_entry& e = entries[i];
        if (e.slot >= uint32_t(t->slots) || e.index >= uint32_t(t->slot_pages) || e.page < -1 || e.page >= t->n_pages)
            fail(GE_ERR_INVALID, "page_table_set: entry %d: slot %u of %d, index %u of %d, page %d of %d (or -1)", i, e.slot, t->slots,
                 e.index, t->slot_pages, e.page, t->n_pages);
        highest = std::max(highest, e.page);
    }
    if (n == 0) return;
    if (size_t(highest) + 1 > t->writer.size()) t->writer.resize(size_t(highest) + 1, 0u);
    auto place = [&](const ge_page_entry& e) { return size_t(e.slot) * size_t(t->slot_pages) + e.index; };
    std::vector<int32_t> before(static_cast<size_t>(n));
    std::vector<uint32_t> again;
    again.reserve(static_cast<size_t>(n));  // nothing can fail once the pages are set
    OpTemps temps(c);
    uint2* const list = reinterpret_cast<uint2*>(op_lists(c, size_t(n) * sizeof(uint2)));
    for (int i = 0; i < n; i++) {
        before[size_t(i)] = t->pages[place(entries[i])];
        t->pages[place(entries[i])] = entries[i].page;
    }
    // of two entries for one place both carry the last one's page
    for (int i = 0; i < n; i++) list[i] = make_uint2(uint32_t(place(entries[i])), uint32_t(t->pages[place(entries[i])]));
    try {
        launch(c, "page_table_set", [&] { return launch_table_set(c->stream, t->dev, list, n); });
        hip_check(hipStreamSynchronize(c->stream), "hipStreamSynchronize");
    } catch (...) {
        for (int i = n; i-- > 0;) t->pages[place(entries[i])] = before[size_t(i)];
        throw;
    }
    // A page behind a slot's last one, the common case, lengthens its run; the runs of slots with any other entry
    // are found again.
    for (int i = 0; i < n; i++) {
        ge_page_table::Run& r = t->runs[entries[i].slot];
        if (entries[i].page >= 0 && int(entries[i].index) == r.end && r.end > 0 && t->pages[place(entries[i])] >= 0)
            r.end++;
        else
            again.push_back(entries[i].slot);
    }
    std::sort(again.begin(), again.end());
    again.erase(std::unique(again.begin(), again.end()), again.end());
    for (const uint32_t slot : again) t->runs[slot] = find_run(t, slot);
}

// ---------------------------------------------------------------------------- attention

constexpr const char* kAttend = "attention_paged";

void attend(ge_ctx* c, const ge_paged_shape* shape, const void* q, const ge_page_table* t, const void* k_pages, const void* v_pages,
            const ge_paged_seq* seqs, int n_seqs, void* out) {
    if (!shape) fail(GE_ERR_INVALID, "%s: null shape", kAttend);
    ge_paged_shape s = *shape;
    if (s.type != GE_TYPE_F16 && s.type != GE_TYPE_BF16) fail(GE_ERR_INVALID, "%s: type %d is neither F16 nor BF16", kAttend, s.type);
    if (!causal_head_dim_ok(s.head_dim)) fail(GE_ERR_INVALID, "%s: head dim %d (64, 128, 256 or 512)", kAttend, s.head_dim);
    if (s.heads <= 0 || s.kv_heads <= 0 || s.heads % s.kv_heads || s.heads > kMaxHeads)
        fail(GE_ERR_INVALID, "%s: %d query heads over %d KV heads (a multiple, up to %d)", kAttend, s.heads, s.kv_heads, kMaxHeads);
    if (s.q_rows < 0 || s.q_rows >= kAttentionMaxRows || s.window < 0 || s.window >= kAttentionMaxRows || n_seqs < 0)
        fail(GE_ERR_INVALID, "%s: query rows and window from 0 to under 2^30, sequences from 0 on", kAttend);
    if (int64_t(s.q_rows) * (s.heads / s.kv_heads) >= kAttentionMaxRows)
        fail(GE_ERR_INVALID, "%s: %d rows of %d query heads a KV head pass 2^30", kAttend, s.q_rows, s.heads / s.kv_heads);
    if (!std::isfinite(s.scale)) fail(GE_ERR_INVALID, "%s: scale is not finite", kAttend);
    if (!(s.cap >= 0.0f && s.cap <= kMaxCap)) fail(GE_ERR_INVALID, "%s: cap %g (0 to 1024)", kAttend, double(s.cap));
    const int64_t q_width = int64_t(s.heads) * s.head_dim;
    check_rows_stride(kAttend, "q", s.q_stride, q_width, 8);
    check_rows_stride(kAttend, "out", s.out_stride, q_width, 8);
    check_table(kAttend, c, t);
    check_page_stride(kAttend, s.page_stride, page_elements(t, s.kv_heads, s.head_dim));
    if (n_seqs == 0) return;
    if (!seqs) fail(GE_ERR_INVALID, "%s: null sequences", kAttend);
    if (check_seqs(kAttend, t, seqs, n_seqs, s.q_rows) == 0) return;
    bool keys = false;
    for (int i = 0; i < n_seqs; i++) {
        const ge_paged_seq& e = seqs[i];
        if (!e.q_len || !e.kv_len) continue;
        keys = true;
        const int64_t low = s.window ? std::max<int64_t>(0, int64_t(e.kv_len) - e.q_len - s.window + 1) : 0;
        if (!has_pages(t, e.slot, low >> t->page_shift, int64_t((e.kv_len - 1) >> t->page_shift) + 1))
            fail(GE_ERR_INVALID, "%s: sequence %d: slot %u lacks a page of keys [%lld, %u)", kAttend, i, e.slot, static_cast<long long>(low), e.kv_len);
    }
    if (!q || !out || (keys && (!k_pages || !v_pages))) fail(GE_ERR_INVALID, "%s: q, out, and the pages of k and v", kAttend);
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(k_pages, 16) || !aligned(v_pages, 16))
        fail(GE_ERR_INVALID, "%s: buffers are 16-byte aligned", kAttend);

    if (!c->paged_ready) {
        hip_check(paged_configure(), "hipFuncSetAttribute");
        c->paged_ready = true;
    }
    const PagedPlan p = plan_paged(s, seqs, n_seqs);
    if (p.workgroups * uint64_t(s.kv_heads) > kCausalMaxGroups || p.joins.size() * uint64_t(s.kv_heads) > kCausalMaxGroups / 4 ||
        p.items.size() >= kDirect || p.part_rows >= kDirect)
        fail(GE_ERR_INVALID, "%s: the call's rows and keys are too many for one call", kAttend);
    OpTemps temps(c);
    PagedInline in;
    CausalInline join_in;
    const bool few = p.items.size() <= size_t(kPagedInlineItems), few_joins = p.joins.size() <= size_t(kCausalInlineJoins);
    const size_t item_bytes = few ? 0 : (p.items.size() * sizeof(PagedItem) + 255) / 256 * 256;
    const size_t join_bytes = few_joins ? 0 : p.joins.size() * sizeof(CausalJoin);
    unsigned char* const lists = item_bytes + join_bytes ? op_lists(c, item_bytes + join_bytes) : nullptr;
    std::copy(p.items.begin(), p.items.end(), few ? in.items : reinterpret_cast<PagedItem*>(lists));
    std::copy(p.joins.begin(), p.joins.end(), few_joins ? join_in.joins : reinterpret_cast<CausalJoin*>(lists + item_bytes));
    const size_t o_at = temps.reserve(p.part_rows * size_t(s.kv_heads) * size_t(s.head_dim) * 4);
    const size_t ml_at = temps.reserve(p.part_rows * size_t(s.kv_heads) * 8);
    unsigned char* const base = p.part_rows ? temps.base() : nullptr;

    PagedArgs a{};
    a.q = static_cast<const uint16_t*>(q);
    a.k = static_cast<const uint16_t*>(k_pages);
    a.v = static_cast<const uint16_t*>(v_pages);
    a.out = static_cast<uint16_t*>(out);
    a.paged_items = few ? nullptr : reinterpret_cast<const PagedItem*>(lists);
    a.joins = few_joins ? nullptr : reinterpret_cast<const CausalJoin*>(lists + item_bytes);
    a.part_o = reinterpret_cast<float*>(base + o_at);
    a.part_ml = reinterpret_cast<float2*>(base + ml_at);
    a.q_stride = s.q_stride;
    a.out_stride = s.out_stride;
    a.part_rows = p.part_rows;
    a.n_items = int(p.workgroups);
    a.n_joins = int(p.joins.size());
    a.join_rows = p.join_rows;
    a.group = s.heads / s.kv_heads;
    a.kv_heads = s.kv_heads;
    a.window = s.window;
    a.q_flip = s.scale < 0.0f ? 0x80008000u : 0u;
    a.table = t->dev;
    a.page_stride = s.page_stride;
    a.slot_pages = t->slot_pages;
    a.page_shift = t->page_shift;
    constexpr float kLog2e = 1.4426950408889634f;
    if (s.cap > 0.0f) {
        a.cap_z = std::min(2 * kLog2e * (std::fabs(s.scale) / s.cap), FLT_MAX);
        a.cap_top = std::max(s.cap * kLog2e, FLT_MIN);
        a.c = 1.0f;
    } else {
        // a hidden key's -inf times this stays -inf, also at scale 0
        a.c = std::min(std::max(std::fabs(s.scale) * kLog2e, FLT_MIN), FLT_MAX);
    }
    launch(c, kAttend, [&] { return launch_paged(c->stream, a, in, s.head_dim, s.type == GE_TYPE_BF16, p.kinds); });
    if (a.n_joins)
        launch(c, "attention_join", [&] {
            // four parts a group of lanes: few rows of many parts
            int split = 1;
            while (split < 16 && p.join_parts > 4 * split) split *= 2;
            return launch_paged_join(c->stream, a, join_in, s.head_dim, s.type == GE_TYPE_BF16, split);
        });
    hip_check(hipStreamSynchronize(c->stream), "hipStreamSynchronize");
}

}  // namespace
}  // namespace ge

using ge::fail;
using ge::guarded;

extern "C" {

int ge_op_rotary_create(ge_ctx* c, const ge_rotary_desc* desc, ge_rotary** out) {
    if (out) *out = nullptr;
    double* turns = nullptr;
    const int rc = guarded(c, [&] {
        if (!desc || !out) fail(GE_ERR_INVALID, "rotary: null description or result");
        ge::check_rotary(*desc);
        std::unique_ptr<ge_rotary> r(new ge_rotary);
        const std::vector<double> t = ge::rotary_turns(*desc);
        turns = static_cast<double*>(ge::dev_alloc(t.size() * 8, "rotary positions"));
        ge::hip_check(hipMemcpy(turns, t.data(), t.size() * 8, hipMemcpyHostToDevice), "hipMemcpy");
        r->ctx = c;
        r->dims = desc->dims;
        r->layout = desc->layout;
        // the sine and cosine times up to 1, the sums times the rest: no product leaves fp32's range on the way
        // to a result that does not
        const float m = desc->magnitude == 0.0f ? 1.0f : desc->magnitude;
        (std::fabs(m) > 1.0f ? r->gain : r->fade) = m;
        r->turns = turns;
        *out = r.release();
    });
    if (rc != GE_OK && turns) (void)hipFree(turns);
    return rc;
}

int ge_op_rotary_destroy(ge_ctx* c, ge_rotary* r) {
    if (!r) return GE_OK;
    return guarded(c, [&] {
        if (r->ctx != c) fail(GE_ERR_INVALID, "rotary: the rotary positions are another context's");
        ge::hip_check(hipFree(r->turns), "hipFree");
        delete r;
    });
}

int ge_op_rotate_heads(ge_ctx* c, const ge_heads_shape* shape, const ge_rotary* rotary, const void* q, const void* k,
                       const void* q_norm, const void* k_norm, const void* positions, void* q_out, void* k_out) {
    return guarded(c, [&] { ge::rotate(c, shape, rotary, q, k, q_norm, k_norm, positions, q_out, k_out); });
}

int ge_op_page_table_create(ge_ctx* c, int32_t slots, int32_t slot_pages, int32_t page_rows, int32_t n_pages, ge_page_table** out) {
    if (out) *out = nullptr;
    int32_t* dev = nullptr;
    const int rc = guarded(c, [&] {
        if (!out) fail(GE_ERR_INVALID, "page table: null result");
        if (page_rows < ge::kPagedAlign || page_rows > ge::kMaxPageRows || (page_rows & (page_rows - 1)))
            fail(GE_ERR_INVALID, "page table: pages of %d rows (a power of two from %d to %d)", page_rows, ge::kPagedAlign, ge::kMaxPageRows);
        if (slots <= 0 || slot_pages <= 0 || int64_t(slots) * slot_pages > ge::kMaxTable)
            fail(GE_ERR_INVALID, "page table: %d slots of %d pages (1 on, together up to 2^28)", slots, slot_pages);
        if (int64_t(slot_pages) * page_rows >= ge::kAttentionMaxRows)
            fail(GE_ERR_INVALID, "page table: %d pages of %d rows pass 2^30", slot_pages, page_rows);
        if (n_pages <= 0 || n_pages > ge::kMaxPages) fail(GE_ERR_INVALID, "page table: %d pages (1 to 2^28)", n_pages);
        std::unique_ptr<ge_page_table> t(new ge_page_table);
        t->ctx = c;
        t->slots = slots;
        t->slot_pages = slot_pages;
        t->page_rows = page_rows;
        t->page_shift = __builtin_ctz(uint32_t(page_rows));
        t->n_pages = n_pages;
        t->pages.assign(size_t(slots) * size_t(slot_pages), -1);
        t->runs.assign(size_t(slots), {0, 0});
        dev = static_cast<int32_t*>(ge::dev_alloc(t->pages.size() * 4, "page table"));
        t->dev = dev;
        *out = t.release();
    });
    if (rc != GE_OK && dev) (void)hipFree(dev);
    return rc;
}

int ge_op_page_table_set(ge_ctx* c, ge_page_table* t, const ge_page_entry* entries, int32_t n) {
    return guarded(c, [&] { ge::set_pages(c, t, entries, n); });
}

int ge_op_page_table_destroy(ge_ctx* c, ge_page_table* t) {
    if (!t) return GE_OK;
    return guarded(c, [&] {
        ge::check_table("page table", c, t);
        ge::hip_check(hipFree(t->dev), "hipFree");
        delete t;
    });
}

int ge_op_paged_append(ge_ctx* c, const ge_heads_shape* shape, const ge_rotary* rotary, const void* q, const void* k,
                       const void* v, const void* q_norm, const void* k_norm, const void* positions, const ge_page_table* table,
                       const ge_paged_seq* seqs, int32_t n_seqs, void* q_out, void* k_pages, void* v_pages) {
    return guarded(c, [&] {
        ge::append(c, shape, rotary, q, k, v, q_norm, k_norm, positions, table, seqs, n_seqs, q_out, k_pages, v_pages);
    });
}

int ge_op_attention_paged(ge_ctx* c, const ge_paged_shape* shape, const void* q, const ge_page_table* table, const void* k_pages,
                          const void* v_pages, const ge_paged_seq* seqs, int32_t n_seqs, void* out) {
    return guarded(c, [&] { ge::attend(c, shape, q, table, k_pages, v_pages, seqs, n_seqs, out); });
}

}  // extern "C"
