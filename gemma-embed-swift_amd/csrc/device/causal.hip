// Attention of causal models: packed prompts and cached keys, and a batch over a shared prefix
// (gfx950). Every query row i of a sequence sees the keys j <= i + shift and, with a window,
// j > i + shift - window:
//   o_i = sum_j exp(scale q_i.k_j) v_j / sum_j exp(scale q_i.k_j),   0 where it sees no key.
//
// Rows. The G = heads / kv_heads query heads of a KV head score against the same keys, so the kernels
// work on stacked rows: row r of a KV head is token r / G of the item's sequence, query head
// kvh G + r % G. Of a batch over a shared prefix the rows of all its sequences stack up too.
//
// One wave holds 32 rows for the whole kernel and streams key blocks past them on
// v_mfma_f32_32x32x16 (twice the rate of the 16x16x32 form here):
//   S^T = K Q^T: A = 32 keys x 16 dims from LDS, B = the rows' fragments in registers. Lane l's 16
//     accumulators are the keys 8 (e / 4) + 4 (l / 32) + e % 4 of row l % 32, so a row's softmax
//     needs one exchange between two lanes.
//   O^T += V^T P^T: the same accumulators, rounded to the inputs' type, are the B operand of the
//     16-key steps when V^T's keys are taken in that order; V^T comes from V's rows in LDS by the
//     transposing LDS read (4 keys x 16 dims a read of 16 lanes), so no transposed copy of V exists.
// The running maximum moves only when a score passes it by 8 (in log2), as in attention.hip. P is taken
// 2^6 higher in fp16, which uses its range up to 2^14 and keeps keys of 2^-30 of the maximum, and 2^32 lower in
// bf16, whose values may themselves be fp32's largest: the sum of 2^24 of them, each 8 above the maximum, stays
// in range, and so do keys of 2^-94 of the maximum over ordinary values. Rounding P to
// the inputs' type (half a step, 2^-11 or 2^-8 of a weight at most) is what the matrix instruction
// takes; the sum of the weights is fp32, of P as rounded, so that a row is a mean of the values it sees: with P
// before rounding, 1 to 3% of the results of values that are all the type's largest were infinite.
//
// Bounds. Long prompts: the matrix instructions, at the clock the card's power leaves them (16384 tokens, 32
// heads of 128 over 8: 2.04 to 2.16 ms, 1.02 to 1.08 PFLOP/s of visible pairs; the pipe 55% busy at 1.6 GHz).
// Single tokens: HBM (48 over caches of up to 8000 keys: 145 us, 5.4 TB/s). Small calls: a chain of reads, the
// item, q and the first keys, and the stores, 6 to 7 us.
#include "causal_rows.hpp"

namespace ge {
namespace {

// The key blocks of an item: those of its prefix keys, then those of its own, none of both.
template <int BK>
struct Span {
    static constexpr int kKeys = BK;
    const CausalArgs& args;
    int own0, blocks;      // the first block of own keys, all blocks
    int lo, end0, skip;    // the item's first key, the end of its prefix keys, the keys that block own0 - 1 lacks
    int hi;
    uint32_t own_row;      // + key: its row of k and v, modulo 2^32

    __device__ __forceinline__ Span(const CausalArgs& a, const CausalItem& it) : args(a), lo(int(it.k_lo)), hi(int(it.k_hi)) {
        end0 = min(max(lo, a.prefix_len), hi);
        own0 = (end0 - lo + BK - 1) / BK;
        skip = own0 * BK - (end0 - lo);
        blocks = own0 + (hi - end0 + BK - 1) / BK;
        own_row = it.key0 - uint32_t(a.prefix_len);
    }
    __device__ __forceinline__ int first(int b) const { return lo + b * BK - (b < own0 ? 0 : skip); }
    __device__ __forceinline__ int end(int b) const { return min(first(b) + BK, b < own0 ? end0 : hi); }
    // Block b's rows of k or v (own, prefix) for one head.
    template <int HD>
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows(int b, const uint16_t* own, const uint16_t* prefix, int64_t stride,
                                                          int kvh) const {
        const bool p = b < own0;
        return KvBlock<HD, BK>::rows_of(p ? prefix : own, uint32_t(first(b)) + (p ? 0u : own_row), stride, kvh * HD, end(b) - first(b));
    }
    // Key `key` of block b's value for one head.
    template <int HD>
    __device__ __forceinline__ const uint16_t* value_row(int b, int key, int kvh) const {
        const uint16_t* const rows = b < own0 ? args.prefix_v : args.v;
        return rows + size_t(uint32_t(key) + (b < own0 ? 0u : own_row)) * size_t(args.v_stride) + size_t(kvh) * HD;
    }
};

// ---------------------------------------------------------------------------- many rows: waves over rows

// 128 rows, 32 a wave; the workgroup's waves copy each key block together, two blocks in LDS. At head dim
// 512 the queries (128 registers) and all accumulators (256) do not fit beside the rest: 64 rows, 32 a
// pair of waves. With two workgroups a CU one's softmax runs beside the other's products; alone on a CU a
// block of 32 keys of head dim 256 takes 1.3 us, its four phases one after another.
template <typename T, int HD>
struct Wide {
    static constexpr int NW = 4, DW = HD > 256 ? 2 : 1, BK = HD <= 128 ? 64 : 32;
    static_assert(NW / DW * 32 == causal_wide_rows(HD), "rows of a wide item");
    using Kv = KvBlock<HD, BK>;
    static constexpr int kLds = 2 * 2 * Kv::kBytes;

    static __device__ __forceinline__ void run(const CausalArgs& a, const CausalItem& it, int kvh, unsigned char* lds) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
        const uint32_t kb_bytes = uint32_t(a.k_stride) * 2, vb_bytes = uint32_t(a.v_stride) * 2;
        static_assert(Kv::kChunks % NW == 0 && (BK / 8) % NW == 0 && NW % 2 == 0, "every wave copies chunks of one key parity");
        uint32_t k_off[BK / 8 / NW], v_off[BK / 8 / NW];
#pragma unroll
        for (int i = 0; i < BK / 8 / NW; i++) {
            k_off[i] = Kv::k_lane(lane, wave & 1, kb_bytes) + uint32_t((wave + i * NW) * 8) * kb_bytes;
            v_off[i] = Kv::v_lane(lane, vb_bytes) + uint32_t((wave + i * NW) * 8) * vb_bytes;
        }
        const Span<BK> span(a, it);
        const int blocks = span.blocks;
        auto issue = [&](int b) {
            unsigned char* const at = lds + (b & 1) * 2 * Kv::kBytes;
            const auto kr = span.template rows<HD>(b, a.k, a.prefix_k, a.k_stride, kvh);
            const auto vr = span.template rows<HD>(b, a.v, a.prefix_v, a.v_stride, kvh);
            Kv::template copies<HD / 64, NW>(kr, at, wave, k_off);
            Kv::template copies<HD / 64, NW>(vr, at + Kv::kBytes, wave, v_off);
        };
        const int r0 = int(it.row0) + wave / DW * 32, n = min(32, int(it.n_rows) - wave / DW * 32);
        Rows<T, HD, DW> w;
        HeldBack<T, HD> held;
        held.init(a, it);
        if (blocks > 0) issue(0);
        if (n > 0) w.init(a, it, kvh, r0, n, wave % DW, lane);
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
            if (b + 1 < blocks) issue(b + 1);
            if (n > 0 && kb <= w.hi_any && kb + BK - 1 >= w.lo_any) {
                typename Rows<T, HD, DW>::template Block<BK> blk;
                u32x4 p[BK / 16];
                blk.scores(w, at, lane);
                blk.softmax(w, kb, span.end(b), a.c, lane, p);
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

// 32 rows; the waves take the key blocks in turn, each through LDS of its own, and join at the end. From head
// dim 256 on pairs of waves take a block together, so that the workgroup's LDS is half as large and
// two fit a CU (at 256; a launch of both kinds of items takes the larger of their LDS: with four waves'
// blocks, 128 KB, 128 texts over a prefix of 8192 took 192 us). A wave alone on its LDS waits for its own
// copies only; pairs meet at the workgroup's barriers.
template <typename T, int HD>
struct Narrow {
    static constexpr int DW = HD > 128 ? 2 : 1, KW = 4 / DW, BK = 32;
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

    static __device__ __forceinline__ void run(const CausalArgs& a, const CausalItem& it, int kvh, unsigned char* lds) {
        const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
        const int kw = wave / DW, dims = wave % DW;
        const uint32_t kb_bytes = uint32_t(a.k_stride) * 2, vb_bytes = uint32_t(a.v_stride) * 2;
        // a wave of a pair copies half of the panels
        constexpr int kPanels = HD / 64 / DW;
        uint32_t k_off[BK / 8], v_off[BK / 8];
#pragma unroll
        for (int i = 0; i < BK / 8; i++) {
            k_off[i] = Kv::k_lane(lane, i & 1, kb_bytes) + uint32_t(i * 8) * kb_bytes + uint32_t(dims * kPanels * 128);
            v_off[i] = Kv::v_lane(lane, vb_bytes) + uint32_t(i * 8) * vb_bytes + uint32_t(dims * kPanels * 128);
        }
        const Span<BK> span(a, it);
        const int blocks = span.blocks;
        unsigned char* const K = lds + kw * kPerKw;
        unsigned char* const V = K + Kv::kBytes;
        auto issue_k = [&](int b) {
            const auto r = span.template rows<HD>(b, a.k, a.prefix_k, a.k_stride, kvh);
            Kv::template copies<kPanels, 1>(r, K + dims * kChunks * 1024, 0, k_off);
        };
        auto issue_v = [&](int b) {
            const auto r = span.template rows<HD>(b, a.v, a.prefix_v, a.v_stride, kvh);
            Kv::template copies<kPanels, 1>(r, V + dims * kChunks * 1024, 0, v_off);
        };
        const int r0 = int(it.row0), n = int(it.n_rows);
        Rows<T, HD, DW> w;
        HeldBack<T, HD> held;
        held.init(a, it);
        if (kw < blocks) {
            issue_k(kw);
            issue_v(kw);
        }
        w.init(a, it, kvh, r0, n, dims, lane);
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
            if (more) issue_k(b + KW);
            if (mine) blk.softmax(w, kb, span.end(b), a.c, lane, p);
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
            if (more) issue_v(b + KW);
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
constexpr int causal_lds() {
    int lds = 0;
    if constexpr ((KINDS & kCausalWide) != 0) lds = Wide<T, HD>::kLds;
    if constexpr ((KINDS & kCausalNarrow) != 0) lds = lds > Narrow<T, HD>::kLds ? lds : Narrow<T, HD>::kLds;
    return lds;
}

template <typename T, int HD, int KINDS>
__global__ __launch_bounds__(256, HD <= 256 ? 2 : 1) void causal_kernel(const CausalArgs a, const CausalInline in) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char causal_lds_mem[];
    // Workgroups go to the 8 XCDs in turn: with the KV head fastest, a head's items share an L2.
    const uint32_t at = blockIdx.x / uint32_t(a.kv_heads);
    const int kvh = int(blockIdx.x % uint32_t(a.kv_heads));
    const CausalItem it = uniform_entry<CausalItem>(a.items, in.items, at);
    if (KINDS == kCausalNarrow || ((KINDS & kCausalNarrow) && it.narrow))
        Narrow<T, HD>::run(a, it, kvh, causal_lds_mem);
    else if constexpr ((KINDS & kCausalWide) != 0)
        Wide<T, HD>::run(a, it, kvh, causal_lds_mem);
}

// ---------------------------------------------------------------------------- joining the parts

// HD / 4 lanes a row (64 at most), so that every load is 16 bytes a lane: the parts' maxima and sums, a lane
// a part, then their rows weighted and added in order. (A wave a row, at head dim 64 4 bytes a lane, took
// 10.6 us to join 32768 rows of 1.5 parts; this way 4.9.)
template <int HD>
constexpr int kJoinLanes = HD < 256 ? HD / 4 : 64;
template <int HD>
constexpr int kJoinRows = 256 / kJoinLanes<HD>;  // of a workgroup
template <typename T, int HD>
__global__ __launch_bounds__(256) void causal_join_kernel(const CausalArgs a, const CausalInline in) {
    constexpr int L = kJoinLanes<HD>, E = HD / (4 * L);  // 16-byte loads a lane of a row
    const int lane = int(threadIdx.x) & (L - 1), group0 = int(threadIdx.x & 63) & ~(L - 1);
    const uint32_t at = blockIdx.x / uint32_t(a.kv_heads), kvh = blockIdx.x % uint32_t(a.kv_heads), g = uint32_t(a.group);
    const CausalJoin jn = uniform_entry<CausalJoin>(a.joins, in.joins, at);
    const uint32_t row = blockIdx.y * kJoinRows<HD> + threadIdx.x / L;
    if (row >= jn.n_rows) return;
    const size_t base = size_t(kvh) * a.part_rows + row;
    const uint32_t parts = jn.splits[0] + jn.splits[1];
    auto place = [&](uint32_t s) {
        return base + (s < jn.splits[0] ? jn.part[0] + size_t(s) * jn.stride[0] : jn.part[1] + size_t(s - jn.splits[0]) * jn.stride[1]);
    };
    auto load = [&](uint32_t s) { return s < parts ? a.part_ml[place(s)] : float2{-INFINITY, 0.0f}; };
    float top = -INFINITY;
    for (uint32_t s = 0; s < parts; s += L) top = fmaxf(top, load(s + lane).x);
#pragma unroll
    for (int x = L / 2; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    float sum = 0.0f;
    float4_t o[E] = {};
    for (uint32_t s0 = 0; s0 < parts; s0 += L) {
        const float2 ml = load(s0 + lane);
        // (a part without a weight adds zeros, or the NaN of an infinite value whose key weighs nothing)
        const float f = ml.x == top ? 1.0f : __builtin_amdgcn_exp2f(ml.x - top);
        sum += ml.y * f;
        const int n = int(min(uint32_t(L), parts - s0));
        for (int i0 = 0; i0 < n; i0 += 4) {  // four parts' loads in flight
            float4_t x[4][E];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < E; e++)
                    x[i][e] = *reinterpret_cast<const float4_t*>(a.part_o + place(s0 + min(i0 + i, n - 1)) * HD + (e * L + lane) * 4);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int k = group0 + min(i0 + i, n - 1);
                const float w = __shfl(f, k, 64);
                const bool none = i0 + i >= n;
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[e][j] = none ? o[e][j] : __builtin_fmaf(x[i][e][j], w, o[e][j]);
            }
        }
    }
#pragma unroll
    for (int x = L / 2; x; x >>= 1) sum += __shfl_xor(sum, x, 64);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint32_t r = jn.row0 + row;
    uint16_t* const out = a.out + (size_t(jn.q_token) + r / g) * size_t(a.out_stride) + (size_t(kvh) * g + r % g) * HD;
#pragma unroll
    for (int e = 0; e < E; e++)
        *reinterpret_cast<u32x2*>(out + (e * L + lane) * 4) =
            u32x2{T::pack(o[e][0] * inv, o[e][1] * inv), T::pack(o[e][2] * inv, o[e][3] * inv)};
}

template <typename T, int HD, int KINDS>
hipError_t run_items(hipStream_t s, const CausalArgs& a, const CausalInline& in) {
    launch_kernel(causal_kernel<T, HD, KINDS>, dim3(uint32_t(a.n_items) * uint32_t(a.kv_heads)), dim3(256), uint32_t(causal_lds<T, HD, KINDS>()), s, a, in);
    return hipGetLastError();
}

template <typename T, int HD>
hipError_t run_kinds(hipStream_t s, const CausalArgs& a, const CausalInline& in, int kinds) {
    switch (kinds) {
        case kCausalWide: return run_items<T, HD, kCausalWide>(s, a, in);
        case kCausalNarrow: return run_items<T, HD, kCausalNarrow>(s, a, in);
        case kCausalWide | kCausalNarrow: return run_items<T, HD, kCausalWide | kCausalNarrow>(s, a, in);
    }
    return hipErrorInvalidValue;
}

template <typename T, int HD>
hipError_t run_join(hipStream_t s, const CausalArgs& a, const CausalInline& in) {
    launch_kernel(causal_join_kernel<T, HD>, dim3(uint32_t(a.n_joins) * uint32_t(a.kv_heads), uint32_t(a.join_rows + kJoinRows<HD> - 1) / kJoinRows<HD>),
                  dim3(256), 0, s, a, in);
    return hipGetLastError();
}

template <typename T, int HD, int KINDS>
hipError_t configure_kinds() {
    constexpr int lds = causal_lds<T, HD, KINDS>();
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    return hipFuncSetAttribute(reinterpret_cast<const void*>(causal_kernel<T, HD, KINDS>),
                               hipFuncAttributeMaxDynamicSharedMemorySize, lds);
}

template <typename T, int HD>
hipError_t configure_hd() {
    hipError_t e = configure_kinds<T, HD, kCausalWide>();
    if (e == hipSuccess) e = configure_kinds<T, HD, kCausalNarrow>();
    if (e == hipSuccess) e = configure_kinds<T, HD, kCausalWide | kCausalNarrow>();
    return e;
}

bool args_ok(const CausalArgs& a, int hd) {
    return causal_head_dim_ok(hd) && a.kv_heads > 0 && a.group > 0 && a.n_items >= 0 && a.n_joins >= 0 && a.join_rows >= 0 && a.join_rows <= 128 &&
           uint64_t(a.n_items) * uint64_t(a.kv_heads) <= kCausalMaxGroups && uint64_t(a.n_joins) * uint64_t(a.kv_heads) <= kCausalMaxGroups;
}

}  // namespace

bool causal_head_dim_ok(int hd) { return hd == 64 || hd == 128 || hd == 256 || hd == 512; }

hipError_t launch_causal(hipStream_t s, const CausalArgs& a, const CausalInline& in, int hd, bool bf16, int kinds) {
    if (!args_ok(a, hd)) return hipErrorInvalidValue;
    if (a.n_items == 0) return hipSuccess;
    switch (hd) {
        case 64: return bf16 ? run_kinds<BF16, 64>(s, a, in, kinds) : run_kinds<F16, 64>(s, a, in, kinds);
        case 128: return bf16 ? run_kinds<BF16, 128>(s, a, in, kinds) : run_kinds<F16, 128>(s, a, in, kinds);
        case 256: return bf16 ? run_kinds<BF16, 256>(s, a, in, kinds) : run_kinds<F16, 256>(s, a, in, kinds);
        default: return bf16 ? run_kinds<BF16, 512>(s, a, in, kinds) : run_kinds<F16, 512>(s, a, in, kinds);
    }
}

hipError_t launch_causal_join(hipStream_t s, const CausalArgs& a, const CausalInline& in, int hd, bool bf16) {
    if (!args_ok(a, hd)) return hipErrorInvalidValue;
    if (a.n_joins == 0) return hipSuccess;
    switch (hd) {
        case 64: return bf16 ? run_join<BF16, 64>(s, a, in) : run_join<F16, 64>(s, a, in);
        case 128: return bf16 ? run_join<BF16, 128>(s, a, in) : run_join<F16, 128>(s, a, in);
        case 256: return bf16 ? run_join<BF16, 256>(s, a, in) : run_join<F16, 256>(s, a, in);
        default: return bf16 ? run_join<BF16, 512>(s, a, in) : run_join<F16, 512>(s, a, in);
    }
}

hipError_t causal_configure() {
    const hipError_t e[8] = {configure_hd<F16, 64>(),  configure_hd<BF16, 64>(),  configure_hd<F16, 128>(), configure_hd<BF16, 128>(),
                             configure_hd<F16, 256>(), configure_hd<BF16, 256>(), configure_hd<F16, 512>(), configure_hd<BF16, 512>()};
    for (const hipError_t x : e)
        if (x != hipSuccess) return x;
    return hipSuccess;
}

}  // namespace ge
