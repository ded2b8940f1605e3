// Attention over pages of keys and values (gfx950): chunks of new tokens and single ones over what is cached
// of their sequences. The definition is causal.hip's,
//   o_i = sum_j exp(s_ij) v_j / sum_j exp(s_ij),  s_ij = scale q_i.k_j or cap tanh(scale q_i.k_j / cap),
// over the keys j <= i + shift and, with a window, j > i + shift - window; 0 where there is none. So are the rows,
// the products and the softmax (causal_rows.hpp); the keys come from pages.
//
// A page holds a KV head's rows side by side, so that 8 keys, what one group of copies takes, are in one page and
// follow each other in memory: each group of 8 has a buffer resource of its own, from its page's 64-bit address and
// as long as its keys, and rows past the sequence's end read as zeros. Page numbers are read into scalar registers.
#include "causal_rows.hpp"
#include "paged.hpp"

namespace ge {
namespace {

// tanh as 1 - 2 / (1 + e^2x), off by 2^-21.5: a third of 2^-24 for the exponential's argument and 2^-25 for itself after
// the slope, twice the reciprocal's 2^-23, the last sum's 2^-24. That moves a score by cap 2^-21.5, a weight by as much of
// itself: 2^-13.5 at a cap of 256, a fifth of fp16's half step. From there on (fine) small arguments take the series
// to x^7, whose error below 1/8 is 2^-29 of x; the rest are off by 2^-18 of themselves.
struct Capped {
    static constexpr bool kCurved = true;
    float z, top;
    uint32_t fine;
    __device__ __forceinline__ void operator()(float16_t& s) const {
        if (top == 0.0f) return;
        if (fine) {
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float x = s[e] * z, x2 = x * x;
                const float series = x * __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, -17.0f / 315, 2.0f / 15), -1.0f / 3), 1.0f);
                s[e] = top * (fabsf(x) < 0.125f ? series : tanh(x));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = top * tanh(s[e] * z);
        }
    }
    static __device__ __forceinline__ float tanh(float x) {
        return __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * 2.8853900817779268f)), 1.0f);
    }
};

// The key blocks of an item.
template <int BK>
struct PagedSpan {
    static constexpr int kKeys = BK;
    typedef const __attribute__((address_space(4))) int32_t* Ids;  // read-only: scalar loads
    const PagedArgs& args;
    Ids ids;  // of the sequence
    int lo, hi, blocks;

    __device__ __forceinline__ PagedSpan(const PagedArgs& a, const CausalItem& it)
        : args(a), ids((Ids)(a.table + size_t(it.key0) * size_t(a.slot_pages))), lo(int(it.k_lo)), hi(int(it.k_hi)),
          blocks((hi - lo + BK - 1) / BK) {}
    __device__ __forceinline__ int first(int b) const { return lo + b * BK; }
    __device__ __forceinline__ int end(int b) const { return min(first(b) + BK, hi); }
    // The page of key `key`; of the last one's from there on (nothing of it is read).
    __device__ __forceinline__ int page(int key) const { return ids[uint32_t(min(key, hi - 1)) >> args.page_shift]; }
    // The 8 keys from `key` on, which are in page `page`, of one head.
    template <int HD>
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows(const uint16_t* pool, int page, int key, int kvh) const {
        const size_t at = size_t(page) * size_t(args.page_stride) + size_t((uint32_t(kvh) << args.page_shift) + (uint32_t(key) & ((1u << args.page_shift) - 1))) * HD;
        return buffer_rsrc(pool + at, uint32_t(min(max(hi - key, 0), 8)) * uint32_t(HD * 2));
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

// As causal.hip's wide items: 128 rows (64 at head dim 512), the waves copy each key block together, two in LDS.
template <typename T, int HD>
struct Wide {
    static constexpr int NW = 4, DW = HD > 256 ? 2 : 1, BK = HD <= 128 ? 64 : 32, NG = BK / 8 / NW;
    static_assert(NW / DW * 32 == causal_wide_rows(HD), "rows of a wide item");
    using Kv = KvBlock<HD, BK>;
    static constexpr int kLds = 2 * 2 * Kv::kBytes;

    static __device__ __forceinline__ void run(const PagedArgs& a, const CausalItem& it, int kvh, unsigned char* lds) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
        static_assert(NG >= 1 && NW % 2 == 0, "every wave copies groups of one key parity");
        const uint32_t k_off = Kv::k_lane(lane, wave & 1, HD * 2), v_off = Kv::v_lane(lane, HD * 2);
        const PagedSpan<BK> span(a, it);
        const int blocks = span.blocks;
        int page[NG];
        auto find = [&](int b) {
#pragma unroll
            for (int i = 0; i < NG; i++) page[i] = span.page(span.first(b) + (wave + i * NW) * 8);
        };
        auto issue = [&](int b) {
            unsigned char* const at = lds + (b & 1) * 2 * Kv::kBytes;
#pragma unroll
            for (int i = 0; i < NG; i++) {
                const int k8 = wave + i * NW, key = span.first(b) + k8 * 8;
                copy_group<HD, BK, HD / 64>(span.template rows<HD>(a.k, page[i], key, kvh), at, k8, k_off);
                copy_group<HD, BK, HD / 64>(span.template rows<HD>(a.v, page[i], key, kvh), at + Kv::kBytes, k8, v_off);
            }
        };
        const int r0 = int(it.row0) + wave / DW * 32, n = min(32, int(it.n_rows) - wave / DW * 32);
        Rows<T, HD, DW> w;
        HeldBack<T, HD> held;
        held.init(a, it);
        if (blocks > 0) {
            find(0);
            issue(0);
            find(1);
        }
        if (n > 0) w.init(a, it, kvh, r0, n, wave % DW, lane);
        const Capped curve{a.cap_z, a.cap_top, a.cap_fine};
        for (int b = 0; b < blocks; b++) {
            const int kb = span.first(b);
            unsigned char* const at = lds + (b & 1) * 2 * Kv::kBytes;
            wait_vmcnt<0>();
            if (held.mixed(kb, BK)) {
#pragma unroll
                for (int i = 0; i < Kv::kChunks / NW; i++)  // the chunks this wave copied
                    held.clear(at + Kv::kBytes + (wave + i * NW) * 1024 + lane * 16);
            }
            wait_lgkmcnt0();
            workgroup_barrier();
            if (b + 1 < blocks) {
                issue(b + 1);
                find(b + 2);
            }
            if (n > 0 && kb <= w.hi_any && kb + BK - 1 >= w.lo_any) {
                typename Rows<T, HD, DW>::template Block<BK> blk;
                u32x4 p[BK / 16];
                blk.scores(w, at, lane);
                blk.softmax(w, kb, span.end(b), a.c, lane, p, curve);
                blk.product(w, at + Kv::kBytes, lane, p);
            }
        }
        __syncthreads();  // no one reads K and V any more
        if (n > 0) {
            constexpr int kSlice = kLds / NW;
            w.l = sum_over_halves(w.l);
            w.template finish_rows<kSlice>(a, it, kvh, r0, n, lane, lds + wave * kSlice);
        }
        held.share(lds);
        if (n > 0 && held.any) held.add(a, it, span, kvh, r0, n, w.d0 * 32, w.DT * 32);
    }
};

// ---------------------------------------------------------------------------- few rows: waves over keys

// As causal.hip's narrow items: 32 rows, the waves (pairs of them from head dim 256 on) take the key blocks in
// turn, each through LDS of its own, and join at the end.
template <typename T, int HD>
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

    static __device__ __forceinline__ void run(const PagedArgs& a, const CausalItem& it, int kvh, unsigned char* lds) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
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
        const Capped curve{a.cap_z, a.cap_top, a.cap_fine};
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
template <typename T, int HD, int KINDS>
constexpr int paged_lds() {
    int lds = 0;
    if constexpr ((KINDS & kCausalWide) != 0) lds = Wide<T, HD>::kLds;
    if constexpr ((KINDS & kCausalNarrow) != 0) lds = lds > Narrow<T, HD>::kLds ? lds : Narrow<T, HD>::kLds;
    return lds;
}

template <typename T, int HD, int KINDS>
__global__ __launch_bounds__(256, HD <= 256 ? 2 : 1) void paged_kernel(const PagedArgs a, const CausalInline in) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char paged_lds_mem[];
    // Workgroups go to the 8 XCDs in turn: with the KV head fastest, a head's items share an L2.
    const uint32_t at = blockIdx.x / uint32_t(a.kv_heads);
    const int kvh = int(blockIdx.x % uint32_t(a.kv_heads));
    const CausalItem it = uniform_entry<CausalItem>(a.items, in.items, at);
    if (KINDS == kCausalNarrow || ((KINDS & kCausalNarrow) && it.narrow))
        Narrow<T, HD>::run(a, it, kvh, paged_lds_mem);
    else if constexpr ((KINDS & kCausalWide) != 0)
        Wide<T, HD>::run(a, it, kvh, paged_lds_mem);
}

template <typename T, int HD, int KINDS>
hipError_t run_items(hipStream_t s, const PagedArgs& a, const CausalInline& in) {
    launch_kernel(paged_kernel<T, HD, KINDS>, dim3(uint32_t(a.n_items) * uint32_t(a.kv_heads)), dim3(256), uint32_t(paged_lds<T, HD, KINDS>()), s, a, in);
    return hipGetLastError();
}

template <typename T, int HD>
hipError_t run_kinds(hipStream_t s, const PagedArgs& a, const CausalInline& in, int kinds) {
    switch (kinds) {
        case kCausalWide: return run_items<T, HD, kCausalWide>(s, a, in);
        case kCausalNarrow: return run_items<T, HD, kCausalNarrow>(s, a, in);
        case kCausalWide | kCausalNarrow: return run_items<T, HD, kCausalWide | kCausalNarrow>(s, a, in);
    }
    return hipErrorInvalidValue;
}

template <typename T, int HD, int KINDS>
hipError_t configure_kinds() {
    constexpr int lds = paged_lds<T, HD, KINDS>();
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    return hipFuncSetAttribute(reinterpret_cast<const void*>(paged_kernel<T, HD, KINDS>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
}

template <typename T, int HD>
hipError_t configure_hd() {
    hipError_t e = configure_kinds<T, HD, kCausalWide>();
    if (e == hipSuccess) e = configure_kinds<T, HD, kCausalNarrow>();
    if (e == hipSuccess) e = configure_kinds<T, HD, kCausalWide | kCausalNarrow>();
    return e;
}

}  // namespace

hipError_t launch_paged(hipStream_t s, const PagedArgs& a, const CausalInline& in, int hd, bool bf16, int kinds) {
    if (!causal_head_dim_ok(hd) || a.kv_heads <= 0 || a.group <= 0 || a.n_items < 0 || a.page_shift < 3 ||
        uint64_t(a.n_items) * uint64_t(a.kv_heads) > kCausalMaxGroups)
        return hipErrorInvalidValue;
    if (a.n_items == 0) return hipSuccess;
    switch (hd) {
        case 64: return bf16 ? run_kinds<BF16, 64>(s, a, in, kinds) : run_kinds<F16, 64>(s, a, in, kinds);
        case 128: return bf16 ? run_kinds<BF16, 128>(s, a, in, kinds) : run_kinds<F16, 128>(s, a, in, kinds);
        case 256: return bf16 ? run_kinds<BF16, 256>(s, a, in, kinds) : run_kinds<F16, 256>(s, a, in, kinds);
        default: return bf16 ? run_kinds<BF16, 512>(s, a, in, kinds) : run_kinds<F16, 512>(s, a, in, kinds);
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
