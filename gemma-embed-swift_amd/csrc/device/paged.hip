// Attention over pages of keys and values (gfx950): chunks of new tokens and single ones over what is cached
// of their sequences. The definition is causal.hip's,
//   o_i = sum_j exp(s_ij) v_j / sum_j exp(s_ij),  s_ij = scale q_i.k_j or cap tanh(scale q_i.k_j / cap),
// over the keys j <= i + shift and, with a window, j > i + shift - window; 0 where there is none. So are the rows,
// the products and the softmax (causal_rows.hpp); the keys come from pages.
//
// A page holds a KV head's rows side by side, so that 8 keys, what one group of copies takes, are in one page and
// follow each other in memory: each group of 8 has a buffer resource of its own, from its page's 64-bit address and
// as long as its keys, and rows past the sequence's end read as zeros. Page numbers are read into scalar registers.
//
// What bounds it, of 1.3 PFLOP/s (a large product) and 7.0 TB/s (reads of one run; 5.9 of 4 KB pieces in no order): long prompts
// at head dim 128 the card's power, the matrix pipe 56% busy at 1.66 GHz (8192 tokens over 16192 keys, 32 heads over 8: 1445
// to 1605 us on several cards, 1.01 to 1.12 PFLOP/s); at head dim 64 exponentials and sums beside the products, the VALU 62%
// and the matrix pipe 41% busy (16 heads over 8: 445 to 520 us, 0.78 to 0.91 PFLOP/s); at 256 the same with 35 and 48% (4 heads
// over 2: 400 and 22 us, 0.97); at 512 one wave a SIMD, beside which nothing runs while it waits: 33 and 25% (4 heads: 1290 us, 0.63).
// Tokens the reads (64 over 100 to 8000 keys, pages of 16: 182 us, 5.5 TB/s). Chunks the few items a CU and the parts they leave
// (5 x 301 to 700 over 2000 to 9700, 16 heads of 64 over 8: 87 to 94 and 9 us, 0.60 to 0.65 PFLOP/s; 3 x 500 to 1500, window 1024, 4 capped
// heads of 256 over 2: 34 and 8 us, of which 15 are keys and 12 the way in and out).
#include "causal_rows.hpp"
#include "paged.hpp"

namespace ge {
namespace {

// tanh as 1 - 2 / (1 + e^2x), off by 2^-21.5: a third of 2^-24 for the exponential's argument and 2^-25 for itself after
// the slope, twice the reciprocal's 2^-23, the last sum's 2^-24. That moves a score by cap 2^-21.5 and a weight by as much
// of itself: 2^-16 at a cap of 50, 2^-11.5 at the largest, 1024. (A series for small arguments would keep larger caps
// exact, at twice the instructions.)
struct Capped {
    static constexpr bool kCurved = true;
    float z, top;  // z: 2 log2(e) scale / cap
    __device__ __forceinline__ float operator()(float s) const {
        return __builtin_fmaf(-2.0f * top, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(s * z)), top);
    }
};
struct Uncapped : Straight {
    __device__ __forceinline__ Uncapped(float, float) {}
    __device__ __forceinline__ float operator()(float s) const { return s; }
};

// The key blocks of an item.
template <int BK>
struct PagedSpan {
    static constexpr int kKeys = BK;
    typedef const __attribute__((address_space(4))) int32_t* Ids;  // read-only: scalar loads
    const PagedArgs& args;
    Ids ids;  // of the sequence
    int lo, hi, blocks;
    uint32_t slot;

    __device__ __forceinline__ PagedSpan(const PagedArgs& a, const CausalItem& it)
        : args(a), ids((Ids)(a.table + size_t(it.key0) * size_t(a.slot_pages))), lo(int(it.k_lo)), hi(int(it.k_hi)),
          blocks((hi - lo + BK - 1) / BK), slot(it.key0) {}
    __device__ __forceinline__ int first(int b) const { return lo + b * BK; }
    __device__ __forceinline__ int end(int b) const { return min(first(b) + BK, hi); }
    // The page of the item's group `group` of 8 keys, a lane's own; 0 past the last.
    __device__ __forceinline__ int group_page(int group) const {
        const int key = lo + group * 8;
        return key < hi ? (args.table + size_t(slot) * size_t(args.slot_pages))[uint32_t(key) >> args.page_shift] : 0;
    }
    // The page of key `key`; of the last one's from there on (nothing of it is read).
    __device__ __forceinline__ int page(int key) const { return ids[uint32_t(min(key, hi - 1)) >> args.page_shift]; }
    // The 8 keys from `key` on, which are in page `page`, of one head.
    template <int HD>
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows(const uint16_t* pool, int page, int key, int kvh) const {
        const size_t at = size_t(page) * size_t(args.page_stride) + size_t((uint32_t(kvh) << args.page_shift) + (uint32_t(key) & ((1u << args.page_shift) - 1))) * HD;
        // (as a scalar: a maximum of a minimum would be one vector instruction, and the resource a loop over its lanes)
        const int keys = __builtin_amdgcn_readfirstlane(min(max(hi - key, 0), 8));
        return buffer_rsrc(pool + at, uint32_t(keys) * uint32_t(HD * 2));
    }
    template <int HD>
    __device__ __forceinline__ const uint16_t* value_row(int, int key, int kvh) const {
        return args.v + size_t(page(key)) * size_t(args.page_stride) +
               size_t((uint32_t(kvh) << args.page_shift) + (uint32_t(key) & ((1u << args.page_shift) - 1))) * HD;
    }
};

// The wave's chunks of panels [0, PANELS) of one group of 8 keys, k8 of its block.
template <int HD, int BK, int PANELS, int P = 0>
__device__ __forceinline__ void copy_group(__amdgpu_buffer_rsrc_t r, unsigned char* block, int k8, uint32_t off) {
    if constexpr (P < PANELS) {
        KvBlock<HD, BK>::template copy<P>(r, block, k8, off);
        copy_group<HD, BK, PANELS, P + 1>(r, block, k8, off);
    }
}

// ---------------------------------------------------------------------------- many rows: waves over rows

// As causal.hip's wide items: 128 rows, 32 a wave (64 at head dim 512, 32 a pair of waves); the waves copy each key
// block together, two in LDS.
template <typename T, int HD, typename CURVE>
struct Wide {
    static constexpr int NW = 4, DW = HD > 256 ? 2 : 1, BK = HD <= 128 ? 64 : 32, NG = BK / 8 / NW;
    static_assert(NW / DW * 32 == paged_wide_rows(HD), "rows of a wide item");
    static_assert(NG >= 1 && NW % 2 == 0, "every wave copies groups of one key parity");
    using Kv = KvBlock<HD, BK>;
    using W = Rows<T, HD, DW, DW>;
    static constexpr int kBlocks = 2 * 2 * Kv::kBytes, kShares = DW > 1 ? BK * 128 : 0;  // a wave's, of the scores
    static constexpr int kLds = kBlocks + NW * kShares;

    static __device__ __forceinline__ void run(const PagedArgs& a, const CausalItem& it, int kvh, int lane, unsigned char* lds) {
        const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
        const uint32_t k_off = Kv::k_lane(lane, wave & 1, HD * 2), v_off = Kv::v_lane(lane, HD * 2);
        const PagedSpan<BK> span(a, it);
        const int blocks = span.blocks;
        // The pages of 64 groups of 8 keys (kAhead blocks) at a time, a lane a group, read when the ones before them are
        // taken. (As scalar loads in every block they cost registers across its branches: at head dim 256 150 spilled.)
        constexpr int kAhead = 64 * 8 / BK;
        int ids = 0, ids_next = span.group_page(lane);
        __amdgpu_buffer_rsrc_t rk[NG], rv[NG];
        auto prepare = [&](int b) {
            if (b % kAhead == 0) {
                ids = ids_next;
                ids_next = span.group_page((b + kAhead) * (BK / 8) + lane);
            }
#pragma unroll
            for (int i = 0; i < NG; i++) {
                const int k8 = wave + i * NW, key = span.first(b) + k8 * 8;
                const int page = __builtin_amdgcn_readlane(ids, b % kAhead * (BK / 8) + k8);
                rk[i] = span.template rows<HD>(a.k, page, key, kvh);
                rv[i] = span.template rows<HD>(a.v, page, key, kvh);
            }
        };
        auto issue = [&](int b) {
            unsigned char* const at = lds + (b & 1) * 2 * Kv::kBytes;
            prepare(b);
#pragma unroll
            for (int i = 0; i < NG; i++) {
                copy_group<HD, BK, HD / 64>(rk[i], at, wave + i * NW, k_off);
                copy_group<HD, BK, HD / 64>(rv[i], at + Kv::kBytes, wave + i * NW, v_off);
            }
        };
        // Issued together, a block's copies keep its products waiting (16 a wave at head dim 512); from head dim 128 on they
        // stand between the products of the block before: 8192 tokens over 16192 keys 1435 us instead of 1520 (4 heads of 512),
        // 466 and 475 (4 of 256 over 2), 1605 and 1614 (32 of 128 over 8), and at 64, with four workgroups a CU, 518 and 516.
        constexpr bool kBetween = HD >= 128;
        // a wave with no rows repeats the item's last
        const int row = wave / DW * 32, n = min(32, int(it.n_rows) - row), r0 = int(it.row0) + row;
        W w;
        HeldBack<T, HD> held;
        held.init(a, it);
        if (blocks > 0) issue(0);
        w.init(a, it, kvh, n > 0 ? r0 : int(it.row0 + it.n_rows) - 1, max(n, 1), wave % DW, lane);
        const CURVE curve{a.cap_z, a.cap_top};
        // Block b has landed everywhere, block b - 1 has been read, and the next one's copies start.
        auto turn = [&](int b, bool copies) {
            wait_vmcnt<0>();
            if (held.mixed(span.first(b), BK)) {
#pragma unroll
                for (int i = 0; i < Kv::kChunks / NW; i++)  // the chunks this wave copied
                    held.clear(lds + (b & 1) * 2 * Kv::kBytes + Kv::kBytes + (wave + i * NW) * 1024 + lane * 16);
            }
            wait_lgkmcnt0();
            workgroup_barrier();
            if (!copies)
                prepare(b + 1);
            else if (b + 1 < blocks)
                issue(b + 1);
        };
        // The blocks of which the wave's rows see a key, in a loop of their own: accumulators that only some turns
        // change cost registers at every join.
        // Of four workgroups a CU the oldest would end when the youngest has done half, and the CU run out of waves: an
        // item's priority falls as it gets on. Head dim 64, 8192 tokens over 16192 keys: 485 us without, 465 with; 5 x 301 to
        // 700 over 2000 to 9700 in parts: 95 and 89. (With two workgroups a CU it gains 1% or loses 4.)
        constexpr bool kFalls = paged_workgroups(HD) > 2;
        const int quarter = blocks / 4 + 1;
        auto fall = [&](int b) {
            if (kFalls && b == quarter) __builtin_amdgcn_s_setprio(2);
            if (kFalls && b == 2 * quarter) __builtin_amdgcn_s_setprio(1);
            if (kFalls && b == 3 * quarter) __builtin_amdgcn_s_setprio(0);
        };
        const int first = min(max((w.lo_any - span.lo) / BK, 0), blocks);
        const int end = n <= 0 || w.hi_any < span.lo ? first : max(first, min(blocks, (w.hi_any - span.lo) / BK + 1));
        int b = 0;
        auto pass = [&](int b) {
            turn(b, true);
            if constexpr (DW > 1) workgroup_barrier();  // the other pair's, in join
        };
        unsigned char* const shares = lds + kBlocks;
        for (; b < first; b++) pass(b);
        for (; b < end; b++) {
            turn(b, !kBetween);
            fall(b);
            // the next block's copies, one at a time between this one's products (past the last block of no bytes)
            unsigned char* const next = lds + ((b + 1) & 1) * 2 * Kv::kBytes;
            auto between = [&](int step, int steps) {
                constexpr int P = HD / 64, C = NG * 2 * P;
                if (!kBetween || step % (steps / C)) return;
                const int c = step / (steps / C), i = c / (2 * P), v = c / P % 2, panel = c % P;
                Kv::copy_panel(v ? rv[i] : rk[i], next + v * Kv::kBytes, wave + i * NW, v ? v_off : k_off, panel);
            };
            unsigned char* const at = lds + (b & 1) * 2 * Kv::kBytes;
            typename W::template Block<BK> blk;
            u32x4 p[BK / 16];
            blk.scores(w, at, lane, between);
            if constexpr (DW > 1) blk.join(shares + wave * kShares, shares + (wave ^ 1) * kShares, lane);
            blk.softmax(w, span.first(b), span.end(b), a.c, lane, p, curve);
            blk.product(w, at + Kv::kBytes, lane, p);
        }
        for (; b < blocks; b++) pass(b);
        wait_vmcnt<0>();  // the copies of no bytes past the last block, which still write LDS
        // No one reads K and V any more. (With its barriers after the rows' stores a wave waited 1.7 us for those to arrive.)
        held.share(lds);
        if (n > 0) {
            constexpr int kSlice = kBlocks / NW;
            w.l = sum_over_halves(w.l);
            w.template finish_rows<kSlice>(a, it, kvh, r0, n, lane, lds + wave * kSlice);
        }
        if (n > 0 && held.any) held.add(a, it, span, kvh, r0, n, w.d0 * 32, w.DT * 32);
    }
};

// ---------------------------------------------------------------------------- few rows: waves over keys

// As causal.hip's narrow items: 32 rows, the waves (pairs of them from head dim 256 on) take the key blocks in
// turn, each through LDS of its own, and join at the end.
template <typename T, int HD, typename CURVE>
struct Narrow {
    static constexpr int DW = HD > 128 ? 2 : 1, KW = 4 / DW, BK = 32, NG = BK / 8;
    using Kv = KvBlock<HD, BK>;
    static constexpr int kChunks = Kv::kChunks / DW;  // a wave's copies of K, and of V
    using Join = JoinKeys<T, HD, DW, KW>;
    static constexpr int kPerKw = 2 * Kv::kBytes;
    static constexpr int kLds = KW * kPerKw > Join::kLds ? KW * kPerKw : Join::kLds;

    static __device__ __forceinline__ void meet() {
        wait_lgkmcnt0();
        if (DW > 1)
            workgroup_barrier();
        else
            asm volatile("" ::: "memory");
    }

    static __device__ __forceinline__ void run(const PagedArgs& a, const CausalItem& it, int kvh, int lane, unsigned char* lds) {
        const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
        const int kw = wave / DW, dims = wave % DW;
        // a wave of a pair copies half of the panels
        constexpr int kPanels = HD / 64 / DW;
        const uint32_t half = uint32_t(dims * kPanels * 128);
        const uint32_t k_off[2] = {Kv::k_lane(lane, 0, HD * 2) + half, Kv::k_lane(lane, 1, HD * 2) + half};
        const uint32_t v_off = Kv::v_lane(lane, HD * 2) + half;
        const PagedSpan<BK> span(a, it);
        const int blocks = span.blocks;
        unsigned char* const K = lds + kw * kPerKw;
        unsigned char* const V = K + Kv::kBytes;
        int page[NG];  // of the block whose K is copied next, or V
        auto find = [&](int b, int (&to)[NG]) {
#pragma unroll
            for (int i = 0; i < NG; i++) to[i] = span.page(span.first(b) + i * 8);
        };
        auto issue_k = [&](int b) {
#pragma unroll
            for (int i = 0; i < NG; i++)
                copy_group<HD, BK, kPanels>(span.template rows<HD>(a.k, page[i], span.first(b) + i * 8, kvh), K + dims * kChunks * 1024, i, k_off[i & 1]);
        };
        auto issue_v = [&](int b) {
#pragma unroll
            for (int i = 0; i < NG; i++)
                copy_group<HD, BK, kPanels>(span.template rows<HD>(a.v, page[i], span.first(b) + i * 8, kvh), V + dims * kChunks * 1024, i, v_off);
        };
        const int r0 = int(it.row0), n = int(it.n_rows);
        Rows<T, HD, DW> w;
        HeldBack<T, HD> held;
        held.init(a, it);
        int next[NG] = {};
        if (kw < blocks) {
            find(kw, page);
            issue_k(kw);
            issue_v(kw);
            find(kw + KW, page);
        }
        w.init(a, it, kvh, r0, n, dims, lane);
        const CURVE curve{a.cap_z, a.cap_top};
        // Waves alone on their LDS leave when their blocks are done; pairs keep meeting until all are.
        for (int b = kw; b - kw < blocks; b += KW) {
            const int kb = span.first(b);
            const bool mine = b < blocks, more = b + KW < blocks;
            if (DW == 1 && !mine) break;
            typename Rows<T, HD, DW>::template Block<BK> blk;
            u32x4 p[BK / 16];
            wait_vmcnt<kChunks>();  // all but V's copies
            meet();
            if (mine) blk.scores(w, K, lane);
            meet();  // K's reads have returned before its next block is copied over it
            if (more) {
                issue_k(b + KW);
                find(b + 2 * KW, next);
            }
            if (mine) blk.softmax(w, kb, span.end(b), a.c, lane, p, curve);
            if (more)
                wait_vmcnt<kChunks>();  // all but the next K's
            else
                wait_vmcnt<0>();
            if (mine && held.mixed(kb, BK)) {
#pragma unroll
                for (int i = 0; i < kChunks; i++) held.clear(V + (dims * kChunks + i) * 1024 + lane * 16);
            }
            meet();
            if (mine) blk.product(w, V, lane, p);
            meet();
            if (more) {
                issue_v(b + KW);
#pragma unroll
                for (int i = 0; i < NG; i++) page[i] = next[i];
            }
        }
        w.l = sum_over_halves(w.l);
        held.share(lds);
        Join::run(w, kw, dims, lane, lds);
        if (kw > 0) return;
        w.finish(a, it, kvh, r0, n, lane);
        if (held.any) held.add(a, it, span, kvh, r0, n, w.d0 * 32, w.DT * 32);
    }
};

// KINDS: the items of the launch, kCausalWide and kCausalNarrow or one of them.
template <typename T, int HD, typename CURVE, int KINDS>
constexpr int paged_lds() {
    int lds = 0;
    if constexpr ((KINDS & kCausalWide) != 0) lds = Wide<T, HD, CURVE>::kLds;
    if constexpr ((KINDS & kCausalNarrow) != 0) lds = lds > Narrow<T, HD, CURVE>::kLds ? lds : Narrow<T, HD, CURVE>::kLds;
    return lds;
}

template <typename T, int HD, typename CURVE, int KINDS>
__global__ __launch_bounds__(256, paged_workgroups(HD)) void paged_kernel(const PagedArgs a, const PagedInline in) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char paged_lds_mem[];
    // Workgroups go to the 8 XCDs in turn: with the KV head fastest, a head's items share an L2.
    uint32_t at = blockIdx.x / uint32_t(a.kv_heads);
    const int kvh = int(blockIdx.x % uint32_t(a.kv_heads));
    for (;;) {
        int lane = int(threadIdx.x & 63);
        asm volatile("" : "+v"(lane));  // what an item makes of it is not kept over the loop, in registers that it needs
        if (paged_workgroups(HD) > 2) __builtin_amdgcn_s_setprio(3);  // Wide lets it fall
        const PagedItem it = uniform_entry<PagedItem>(a.paged_items, in.items, at);
        if (KINDS == kCausalNarrow || ((KINDS & kCausalNarrow) && it.narrow))
            Narrow<T, HD, CURVE>::run(a, it, kvh, lane, paged_lds_mem);
        else if constexpr ((KINDS & kCausalWide) != 0)
            Wide<T, HD, CURVE>::run(a, it, kvh, lane, paged_lds_mem);
        at = it.next;
        if (at == 0) break;
        wait_lgkmcnt0();
        workgroup_barrier();  // no one reads the item's LDS any more
    }
}

// ---------------------------------------------------------------------------- joining many parts

// Rows of few tiles that end in many parts (a token over a long cache: 64). causal.hip's join has a group of HD / 4
// lanes (64 at most) take a row's parts one after another, which then is the launch's time; here `split` groups of
// the workgroup take a row's parts in turn and add up through LDS, in one order. 4 rows a KV head of 64 parts
// (head dim 128, 8 KV heads): 9.7 us there, 4.0 here. From head dim 256 on, where a wave is a group, rows of more than four
// take 1024 threads; others, and smaller head dims, 256 (128 rows of 41 tiles in 3 parts at head dim 256: 8.7 us, with
// 1024 10.0; 64 parts at head dim 128 4.0 and 4.4).
template <int HD>
constexpr int kJoinLanes = HD < 256 ? HD / 4 : 64;
template <int HD>
constexpr int kJoinGroups(int threads) {
    return threads / kJoinLanes<HD>;
}
template <typename T, int HD, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_join_kernel(const CausalArgs a, const CausalInline in, int split) {
    constexpr int L = kJoinLanes<HD>, G = kJoinGroups<HD>(THREADS), E = HD / (4 * L);  // lanes of a group, groups, 16-byte loads a lane of a row
    __shared__ float4_t lds_o[G][E][L];
    __shared__ float2 lds_ml[G];
    const int lane = int(threadIdx.x) & (L - 1), group = int(threadIdx.x) / L, turn = group & (split - 1);
    const uint32_t at = blockIdx.x / uint32_t(a.kv_heads), kvh = blockIdx.x % uint32_t(a.kv_heads), g = uint32_t(a.group);
    const CausalJoin jn = uniform_entry<CausalJoin>(a.joins, in.joins, at);
    const uint32_t row = blockIdx.y * uint32_t(G / split) + uint32_t(group / split);
    const bool here = row < jn.n_rows;
    const size_t first = size_t(kvh) * a.part_rows + jn.part[0] + (here ? row : 0);
    const uint32_t parts = jn.splits[0];
    float m = -INFINITY, l = 0.0f;
    float4_t o[E] = {};
    for (uint32_t s0 = uint32_t(turn); s0 < parts; s0 += uint32_t(4 * split)) {  // four parts' loads in flight
        float4_t x[4][E];
        float2 ml[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t s = s0 + uint32_t(i * split);
            const size_t r = first + size_t(min(s, parts - 1)) * jn.stride[0];
            ml[i] = s < parts ? a.part_ml[r] : float2{-INFINITY, 0.0f};
#pragma unroll
            for (int e = 0; e < E; e++) x[i][e] = *reinterpret_cast<const float4_t*>(a.part_o + r * HD + (e * L + lane) * 4);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < 4; i++) top = fmaxf(top, ml[i].x);
        const float fade = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
        l *= fade;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] *= fade;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // (a part without a weight adds zeros, or the NaN of an infinite value whose key weighs nothing)
            if (s0 + uint32_t(i * split) >= parts) continue;
            const float f = ml[i].x == top ? 1.0f : __builtin_amdgcn_exp2f(ml[i].x - top);
            l = __builtin_fmaf(ml[i].y, f, l);
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[e][j] = __builtin_fmaf(x[i][e][j], f, o[e][j]);
        }
        m = top;
    }
#pragma unroll
    for (int e = 0; e < E; e++) lds_o[group][e][lane] = o[e];
    if (lane == 0) lds_ml[group] = float2{m, l};
    __syncthreads();
    if (!here || turn) return;
    float top = -INFINITY;
    for (int i = 0; i < split; i++) top = fmaxf(top, lds_ml[group + i].x);
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = float4_t{};
    for (int i = 0; i < split; i++) {
        const float2 ml = lds_ml[group + i];
        const float f = ml.x == top ? 1.0f : __builtin_amdgcn_exp2f(ml.x - top);
        sum = __builtin_fmaf(ml.y, f, sum);
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[e][j] = __builtin_fmaf(lds_o[group + i][e][lane][j], f, o[e][j]);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t r = jn.row0 + row;
    uint16_t* const out = a.out + (size_t(jn.q_token) + r / g) * size_t(a.out_stride) + (size_t(kvh) * g + r % g) * HD;
#pragma unroll
    for (int e = 0; e < E; e++)
        *reinterpret_cast<u32x2*>(out + (e * L + lane) * 4) =
            u32x2{T::pack(o[e][0] * inv, o[e][1] * inv), T::pack(o[e][2] * inv, o[e][3] * inv)};
}

template <typename T, int HD, int THREADS>
hipError_t run_join_of(hipStream_t s, const CausalArgs& a, const CausalInline& in, int split) {
    const int rows = kJoinGroups<HD>(THREADS) / split;
    launch_kernel(paged_join_kernel<T, HD, THREADS>, dim3(uint32_t(a.n_joins) * uint32_t(a.kv_heads), uint32_t(a.join_rows + rows - 1) / uint32_t(rows)),
                  dim3(THREADS), 0, s, a, in, split);
    return hipGetLastError();
}

template <typename T, int HD>
hipError_t run_join(hipStream_t s, const CausalArgs& a, const CausalInline& in, int split) {
    constexpr int groups = kJoinGroups<HD>(256);
    if constexpr (HD >= 256)
        if (split > groups) return run_join_of<T, HD, 1024>(s, a, in, split);
    return run_join_of<T, HD, 256>(s, a, in, split < groups ? split : groups);
}

template <typename T, int HD, typename CURVE, int KINDS>
hipError_t run_items(hipStream_t s, const PagedArgs& a, const PagedInline& in) {
    launch_kernel(paged_kernel<T, HD, CURVE, KINDS>, dim3(uint32_t(a.n_items) * uint32_t(a.kv_heads)), dim3(256), uint32_t(paged_lds<T, HD, CURVE, KINDS>()), s, a, in);
    return hipGetLastError();
}

template <typename T, int HD, typename CURVE>
hipError_t run_kinds(hipStream_t s, const PagedArgs& a, const PagedInline& in, int kinds) {
    switch (kinds) {
        case kCausalWide: return run_items<T, HD, CURVE, kCausalWide>(s, a, in);
        case kCausalNarrow: return run_items<T, HD, CURVE, kCausalNarrow>(s, a, in);
        case kCausalWide | kCausalNarrow: return run_items<T, HD, CURVE, kCausalWide | kCausalNarrow>(s, a, in);
    }
    return hipErrorInvalidValue;
}

template <typename T, int HD, typename CURVE, int KINDS>
hipError_t configure_kinds() {
    constexpr int lds = paged_lds<T, HD, CURVE, KINDS>();
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    return hipFuncSetAttribute(reinterpret_cast<const void*>(paged_kernel<T, HD, CURVE, KINDS>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
}

template <typename T, int HD, typename CURVE>
hipError_t configure_curve() {
    hipError_t e = configure_kinds<T, HD, CURVE, kCausalWide>();
    if (e == hipSuccess) e = configure_kinds<T, HD, CURVE, kCausalNarrow>();
    if (e == hipSuccess) e = configure_kinds<T, HD, CURVE, kCausalWide | kCausalNarrow>();
    return e;
}

template <typename T, int HD>
hipError_t run_head(hipStream_t s, const PagedArgs& a, const PagedInline& in, int kinds) {
    return a.cap_top == 0.0f ? run_kinds<T, HD, Uncapped>(s, a, in, kinds) : run_kinds<T, HD, Capped>(s, a, in, kinds);
}

template <typename T, int HD>
hipError_t configure_hd() {
    const hipError_t e = configure_curve<T, HD, Uncapped>();
    return e == hipSuccess ? configure_curve<T, HD, Capped>() : e;
}

}  // namespace

hipError_t launch_paged(hipStream_t s, const PagedArgs& a, const PagedInline& in, int hd, bool bf16, int kinds) {
    if (!causal_head_dim_ok(hd) || a.kv_heads <= 0 || a.group <= 0 || a.n_items < 0 || a.page_shift < 3 ||
        uint64_t(a.n_items) * uint64_t(a.kv_heads) > kCausalMaxGroups)
        return hipErrorInvalidValue;
    if (a.n_items == 0) return hipSuccess;
    switch (hd) {
        case 64: return bf16 ? run_head<BF16, 64>(s, a, in, kinds) : run_head<F16, 64>(s, a, in, kinds);
        case 128: return bf16 ? run_head<BF16, 128>(s, a, in, kinds) : run_head<F16, 128>(s, a, in, kinds);
        case 256: return bf16 ? run_head<BF16, 256>(s, a, in, kinds) : run_head<F16, 256>(s, a, in, kinds);
        default: return bf16 ? run_head<BF16, 512>(s, a, in, kinds) : run_head<F16, 512>(s, a, in, kinds);
    }
}

hipError_t launch_paged_join(hipStream_t s, const CausalArgs& a, const CausalInline& in, int hd, bool bf16, int split) {
    if (!causal_head_dim_ok(hd) || a.kv_heads <= 0 || a.n_joins < 0 || a.join_rows < 0 || split < 1 || (split & (split - 1)) ||
        uint64_t(a.n_joins) * uint64_t(a.kv_heads) > kCausalMaxGroups / 4)  // up to 1024 threads
        return hipErrorInvalidValue;
    if (a.n_joins == 0) return hipSuccess;
    switch (hd) {
        case 64: return bf16 ? run_join<BF16, 64>(s, a, in, split) : run_join<F16, 64>(s, a, in, split);
        case 128: return bf16 ? run_join<BF16, 128>(s, a, in, split) : run_join<F16, 128>(s, a, in, split);
        case 256: return bf16 ? run_join<BF16, 256>(s, a, in, split) : run_join<F16, 256>(s, a, in, split);
        default: return bf16 ? run_join<BF16, 512>(s, a, in, split) : run_join<F16, 512>(s, a, in, split);
    }
}

hipError_t paged_configure() {
    const hipError_t e[8] = {configure_hd<F16, 64>(),  configure_hd<BF16, 64>(),  configure_hd<F16, 128>(), configure_hd<BF16, 128>(),
                             configure_hd<F16, 256>(), configure_hd<BF16, 256>(), configure_hd<F16, 512>(), configure_hd<BF16, 512>()};
    for (const hipError_t x : e)
        if (x != hipSuccess) return x;
    return hipSuccess;
}

}  // namespace ge
