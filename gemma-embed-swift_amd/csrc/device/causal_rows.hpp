// What the kernels of causal attention are built from (causal.hip, paged.hip): a block of keys and values in
// LDS, 32 rows of queries a wave over it, values that hidden keys hold back, and the join of waves that took
// different keys.
#pragma once

#include "causal.hpp"
#include "half_types.hpp"

namespace ge {
namespace {

constexpr float kLazy = 8.0f;        // the maximum moves when a score passes it by this much (log2)
constexpr int kNoWindow = -(1 << 30);

// Max and sum over lanes l and l ^ 32 (the two halves of a row's keys).
__device__ __forceinline__ float max_over_halves(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_over_halves(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

__device__ __forceinline__ u32x2 lds_read_transposed(const unsigned char* p) {
    return __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_t*)p));
}

// A block of BK keys of one KV head in LDS: K, then V, each in 1 KB chunks of 8 keys x 64 dims (one
// buffer_load ... lds each, eight whole 128-byte lines), chunk (panel, key / 8) at
// (panel BK / 8 + key / 8) KB:
//   K: key k's 16-byte piece c of the panel at 128 (k % 8) + 16 (c ^ (k / 2) % 8): the 16 keys a
//     fragment read takes at a time fall on 16 different 16-byte columns of the 64 banks.
//   V: 128-byte tiles of 4 keys x 16 dims, the source of one transposing read.
template <int HD, int BK>
struct KvBlock {
    static constexpr int kBytes = BK * HD * 2, kChunks = kBytes / 1024;

    // This lane's byte offsets into a chunk's rows of K and V. parity: of the chunk's key / 8.
    static __device__ __forceinline__ uint32_t k_lane(int lane, int parity, uint32_t row_bytes) {
        const int piece = (lane & 7) ^ (parity * 4 + (lane >> 4));
        return uint32_t(lane >> 3) * row_bytes + uint32_t(piece * 16);
    }
    static __device__ __forceinline__ uint32_t v_lane(int lane, uint32_t row_bytes) {
        const int tile = lane >> 3, key = (tile >> 2) * 4 + ((lane & 7) >> 1), dim = (tile & 3) * 16 + (lane & 1) * 8;
        return uint32_t(key) * row_bytes + uint32_t(dim * 2);
    }
    // Chunk (PANEL, k8) of a block whose rows start at r's base; off: the lane's offset of row 8 k8. Rows past
    // r's size read as zeros. The panel goes into the instruction's offset, which moves the LDS address as well
    // as the source's, so that a wave's chunks of a row group share one offset register. (Not into the scalar offset: that
    // one is no part of what is compared with r's size, and taken off it the size of a resource of no rows would be negative.)
    template <int PANEL>
    static __device__ __forceinline__ void copy(__amdgpu_buffer_rsrc_t r, unsigned char* block, int k8, uint32_t off) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            r, (__attribute__((address_space(3))) void*)(block + (PANEL * (BK / 8) + k8) * 1024 - PANEL * 128), 16, off, 0, PANEL * 128, 0);
    }
    // The same for a panel that is a constant once its loop is unrolled.
    template <int PANEL = 0>
    static __device__ __forceinline__ void copy_panel(__amdgpu_buffer_rsrc_t r, unsigned char* block, int k8, uint32_t off, int panel) {
        if (panel == PANEL)
            copy<PANEL>(r, block, k8, off);
        else if constexpr (PANEL + 1 < HD / 64)
            copy_panel<PANEL + 1>(r, block, k8, off, panel);
    }
    // The wave's chunks of panels [0, PANELS) and row groups k8, k8 + STEP, ... in this order.
    template <int PANELS, int STEP, int I = 0>
    static __device__ __forceinline__ void copies(__amdgpu_buffer_rsrc_t r, unsigned char* block, int k8,
                                                  const uint32_t (&off)[BK / 8 / STEP]) {
        constexpr int N = BK / 8 / STEP;
        if constexpr (I < PANELS * N) {
            copy<I / N>(r, block, k8 + I % N * STEP, off[I % N]);
            copies<PANELS, STEP, I + 1>(r, block, k8, off);
        }
    }
    // Rows [key, key + rows) of a tensor whose row 0 is at base, for the head at element offset `at`.
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const uint16_t* base, size_t key, int64_t stride, int at,
                                                                     int rows) {
        return buffer_rsrc(base + key * size_t(stride) + at, uint32_t((rows - 1) * stride + HD) * 2u);
    }
};

// Fragments read ahead of their products (four spill at head dim 256).
template <int HD>
constexpr int kFragmentsAhead = HD == 256 ? 3 : 4;

// What is done between a score's products: nothing.
struct Nothing {
    __device__ __forceinline__ void operator()(int, int) const {}
};

// What becomes of a score besides its factor: nothing.
struct Straight {
    static constexpr bool kCurved = false;
};

// 32 rows of one KV head: queries in registers, accumulators, running maximum and sum. DW waves can hold
// the same rows: they all compute the scores, or each its share's sums of them (QW = DW), which they then add up
// (Block::join), and each takes its share of the head's dims in the product.
template <typename T, int HD, int DW, int QW = 1>
struct Rows {
    static constexpr int KS = HD / 16 / QW, DT = HD / 32 / DW;
    u32x4 q[KS];
    float16_t o[DT];
    float m, l;
    int hi, lo;            // the last and first key this lane's row sees
    int hi_all, hi_any;    // the last key the wave's first row sees (so all do), and its last row
    int lo_all, lo_any;    // the first key the wave's last row sees (so all do), and its first row
    int d0;                // the first 32-dim tile of this wave's accumulators

    // Stacked rows [r0, r0 + n) of the item (n >= 1 rows of this wave; lanes past them repeat the last).
    __device__ __forceinline__ void init(const CausalArgs& a, const CausalItem& it, int kvh, int r0, int n, int dims, int lane) {
        const uint32_t r = uint32_t(r0) + uint32_t(min(lane & 31, n - 1)), g = uint32_t(a.group);
        const uint32_t i = r / g, head = uint32_t(kvh) * g + r % g;
        const uint16_t* p = a.q + (size_t(it.q_token) + i) * size_t(a.q_stride) + size_t(head) * HD + (QW > 1 ? dims * (HD / QW) : 0) + (lane >> 5) * 8;
#pragma unroll
        for (int s = 0; s < KS; s++) q[s] = *reinterpret_cast<const u32x4*>(p + s * 16) ^ a.q_flip;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = float16_t{};
        m = -INFINITY;
        l = 0.0f;
        d0 = dims * DT;
        const int last = int(it.k_hi) - 1, first = a.window ? it.shift - a.window + 1 : kNoWindow;
        const int i0 = int(uint32_t(r0) / g), i1 = int(uint32_t(r0 + n - 1) / g);
        hi = min(int(i) + it.shift, last);
        lo = int(i) + first;
        hi_all = min(i0 + it.shift, last);
        hi_any = min(i1 + it.shift, last);
        lo_all = i1 + first;
        lo_any = i0 + first;
    }

    // One block of BK keys from index kb on, in LDS at K and V.
    template <int BK>
    struct Block {
        static constexpr int KT = BK / 32, kAhead = kFragmentsAhead<HD>;
        float16_t s[KT];

        // between(step, steps) stands before each step's product.
        template <typename BETWEEN = Nothing>
        __device__ __forceinline__ void scores(const Rows& w, const unsigned char* K, int lane, const BETWEEN& between = {}) {
            const int key = lane & 31, f = (key >> 1) & 7;
            const unsigned char* at[4];
#pragma unroll
            for (int c = 0; c < 4; c++) at[c] = K + (QW > 1 ? w.d0 / 2 * (BK * 128) : 0) + key * 128 + (((2 * c + (lane >> 5)) ^ f) * 16);
            // fragments read kAhead steps before their product; the barriers keep the scheduler from
            // reading all of them first, which spills
            u32x4 ring[kAhead];
            auto read = [&](int i) {
                const int t = i / KS, k = i % KS;
                ring[i % kAhead] = *reinterpret_cast<const u32x4*>(at[k & 3] + (k >> 2) * (BK * 128) + t * 4096);
            };
#pragma unroll
            for (int i = 0; i < kAhead; i++) read(i);
#pragma unroll
            for (int i = 0; i < KT * KS; i++) {
                const int t = i / KS, k = i % KS;
                if (k == 0) s[t] = float16_t{};
                __builtin_amdgcn_sched_barrier(0);
                between(i, KT * KS);
                s[t] = T::mfma(ring[i % kAhead], w.q[k], s[t]);
                if (i + kAhead < KT * KS) read(i + kAhead);
            }
        }

        // The shares' sums, through 1024 KT floats of LDS a wave: `mine` and the other wave's of a pair.
        __device__ __forceinline__ void join(unsigned char* mine, const unsigned char* other, int lane) {
            static_assert(QW == 1 || QW == 2, "pairs");
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4_t*>(mine + (t * 4 + e / 4) * 1024 + lane * 16) = float4_t{s[t][e], s[t][e + 1], s[t][e + 2], s[t][e + 3]};
            wait_lgkmcnt0();
            workgroup_barrier();
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4_t x = *reinterpret_cast<const float4_t*>(other + (t * 4 + e / 4) * 1024 + lane * 16);
#pragma unroll
                    for (int i = 0; i < 4; i++) s[t][e + i] += x[i];
                }
        }

        __device__ __forceinline__ bool sees_all(const Rows& w, int kb, int end) const {
            return kb + BK <= end && kb + BK - 1 <= w.hi_all && kb >= w.lo_all;
        }

        // Hidden keys and those from `end` on to -inf, the running maximum, and P. c: the scores' factor, log2(e) in
        // it; a curve takes the scores before, its factor in it.
        template <typename CURVE = Straight>
        __device__ __forceinline__ void softmax(Rows& w, int kb, int end, float c, int lane, u32x4 (&p)[2 * KT], CURVE curve = {}) {
            if constexpr (CURVE::kCurved) {
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) s[t][e] = curve(s[t][e]);
            }
            if (!sees_all(w, kb, end)) {
                const int k0 = kb + (lane >> 5) * 4, hi = min(w.hi, end - 1);
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int key = k0 + 32 * t + 8 * (e >> 2) + (e & 3);
                        s[t][e] = key <= hi && key >= w.lo ? s[t][e] : -INFINITY;
                    }
            }
            float top = s[0][0];
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) top = fmaxf(top, s[t][e]);
            if (__builtin_amdgcn_ballot_w64(top * c > w.m + kLazy)) {
                // a row's own scores decide, so its bits do not depend on the wave's other rows
                const float block = max_over_halves(top) * c, m_new = block > w.m + kLazy ? block : w.m;
                const float fade = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(w.m - m_new);
                w.l *= fade;
#pragma unroll
                for (int d = 0; d < DT; d++) w.o[d] *= fade;
                w.m = m_new;
            }
            const float ref = w.m == -INFINITY ? 0.0f : T::kRaise - w.m;
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) s[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], c, ref));
            float sum = 0.0f;
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const uint32_t pair = T::pack(s[t][e], s[t][e + 1]);
                    p[2 * t + e / 8][(e % 8) / 2] = pair;
                    sum = T::add(pair, sum);
                }
            w.l += sum;
        }

        // V^T's fragment of 32 dims d and 16 keys t: keys 16 t + 8 j + 4 (lane / 32) + [0, 4) at slots 4 j.
        static __device__ __forceinline__ u32x4 v_fragment(const unsigned char* V, int d, int t) {
            const unsigned char* p = V + ((d >> 1) * (BK / 8) + 2 * t) * 1024 + (d & 1) * 256;
            const u32x2 a = lds_read_transposed(p), b = lds_read_transposed(p + 1024);
            return u32x4{a[0], a[1], b[0], b[1]};
        }

        __device__ __forceinline__ void product(Rows& w, const unsigned char* V, int lane, const u32x4 (&p)[2 * KT]) {
            const unsigned char* vl = V + (w.d0 >> 1) * (BK / 8) * 1024 + (lane >> 5) * 512 + ((lane >> 4) & 1) * 128 + (lane & 15) * 8;
            u32x4 ring[kAhead];
            auto read = [&](int i) { ring[i % kAhead] = v_fragment(vl, i % DT, i / DT); };
#pragma unroll
            for (int i = 0; i < kAhead; i++) read(i);
#pragma unroll
            for (int i = 0; i < 2 * KT * DT; i++) {
                __builtin_amdgcn_sched_barrier(0);
                w.o[i % DT] = T::mfma(ring[i % kAhead], p[i / DT], w.o[i % DT]);
                if (i + kAhead < 2 * KT * DT) read(i + kAhead);
            }
        }
    };

    // Rows to out, or as unnormalised fp32 with their maximum and sum to the partial rows.
    __device__ __forceinline__ void finish(const CausalArgs& a, const CausalItem& it, int kvh, int r0, int n, int lane) {
        const int row = lane & 31, half = lane >> 5;
        if (row >= n) return;
        if (it.part == kDirect) {
            const uint32_t r = uint32_t(r0 + row), g = uint32_t(a.group);
            uint16_t* p = a.out + (size_t(it.q_token) + r / g) * size_t(a.out_stride) +
                          (size_t(kvh) * g + r % g) * HD + d0 * 32 + half * 4;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<u32x2*>(p + 32 * d + 2 * e) =
                        u32x2{T::pack(o[d][e] * inv, o[d][e + 1] * inv), T::pack(o[d][e + 2] * inv, o[d][e + 3] * inv)};
        } else {
            const size_t at = size_t(kvh) * a.part_rows + it.part + uint32_t(r0 - int(it.row0) + row);
            float* p = a.part_o + at * HD + d0 * 32 + half * 4;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4_t*>(p + 32 * d + 2 * e) = float4_t{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
            if (half == 0 && d0 == 0) a.part_ml[at] = float2{m, l};
        }
    }

    // The same through this wave's slice of LDS, where a row's pieces come together: whole 16-byte pieces of a
    // row go out side by side. Straight from the accumulators a store's lanes are all in different rows, and
    // the stores of an item of head dim 256 took 2.4 to 3.4 us.
    template <int SLICE>
    __device__ __forceinline__ void finish_rows(const CausalArgs& a, const CausalItem& it, int kvh, int r0, int n, int lane,
                                                unsigned char* slice) {
        const int row = lane & 31, half = lane >> 5;
        if (it.part == kDirect) {
            constexpr int ROW = DT * 64, P = ROW / 16;  // bytes and pieces of a row
            static_assert(32 * ROW <= SLICE, "a slice holds the rows");
            const uint32_t r = uint32_t(r0 + min(row, n - 1)), g = uint32_t(a.group);
            const size_t at = ((size_t(it.q_token) + r / g) * size_t(a.out_stride) + (size_t(kvh) * g + r % g) * HD + d0 * 32) * 2;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<u32x2*>(slice + row * ROW + (((4 * d + e / 4) ^ (row & (P - 1))) * 16) + half * 8) =
                        u32x2{T::pack(o[d][e] * inv, o[d][e + 1] * inv), T::pack(o[d][e + 2] * inv, o[d][e + 3] * inv)};
#pragma unroll
            for (int i = 0; i < 32 * P / 64; i++) {
                const int x = (i * 64 + lane) / P, c = (i * 64 + lane) % P;
                const size_t row_at = size_t(uint32_t(__shfl(int(uint32_t(at)), x, 64))) | size_t(uint32_t(__shfl(int(uint32_t(at >> 32)), x, 64))) << 32;
                const u32x4 v = *reinterpret_cast<const u32x4*>(slice + x * ROW + ((c ^ (x & (P - 1))) * 16));
                if (x < n) *reinterpret_cast<u32x4*>(reinterpret_cast<unsigned char*>(a.out) + row_at + c * 16) = v;
            }
        } else {
            constexpr int D = 32 * DT * 128 <= SLICE ? DT : SLICE / (32 * 128), ROW = D * 128, P = ROW / 16;  // D dim tiles at a time
            static_assert(DT % D == 0, "whole passes");
            const size_t at = size_t(kvh) * a.part_rows + it.part + uint32_t(r0 - int(it.row0));
            if (lane < n && d0 == 0) a.part_ml[at + row] = float2{m, l};
#pragma unroll
            for (int p = 0; p < DT; p += D) {
#pragma unroll
                for (int d = 0; d < D; d++)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<float4_t*>(slice + row * ROW + (((8 * d + e / 2 + half) ^ (row & 31 & (P - 1))) * 16)) =
                            float4_t{o[p + d][e], o[p + d][e + 1], o[p + d][e + 2], o[p + d][e + 3]};
#pragma unroll 4
                for (int i = 0; i < 32 * P / 64; i++) {
                    const int x = (i * 64 + lane) / P, c = (i * 64 + lane) % P;
                    const u32x4 v = *reinterpret_cast<const u32x4*>(slice + x * ROW + ((c ^ (x & 31 & (P - 1))) * 16));
                    if (x < n) *reinterpret_cast<u32x4*>(a.part_o + (at + x) * HD + (d0 + p) * 32 + c * 4) = v;
                }
            }
        }
    }
};

// A hidden key's P is 0, which its V, where that is infinite or NaN, would still turn into NaN. Only blocks
// with a key that some of the item's rows do not see can hold such a key. Their V is cleared of
// such values by the wave that copied them, before anyone reads it; if there were any, they are added at
// the end to the stored results of the rows that see them, where inf + -inf and NaN come out as in the sum.
template <typename T, int HD>
struct HeldBack {
    int hi_all, hi_any, lo_all, lo_any;  // last and first key that all and that any of the item's rows see
    bool any;

    __device__ __forceinline__ void init(const CausalArgs& a, const CausalItem& it) {
        const uint32_t g = uint32_t(a.group);
        const int i0 = int(it.row0 / g), i1 = int((it.row0 + it.n_rows - 1) / g), last = int(it.k_hi) - 1;
        hi_all = min(i0 + it.shift, last);
        hi_any = min(i1 + it.shift, last);
        const int first = a.window ? it.shift - a.window + 1 : kNoWindow;
        lo_all = i1 + first;
        lo_any = i0 + first;
        any = false;
    }
    __device__ __forceinline__ bool mixed(int kb, int bk) const {
        return (kb + bk - 1 > hi_all && hi_all < hi_any) || kb < lo_all;
    }
    // This lane's 16 bytes of a landed copy.
    __device__ __forceinline__ void clear(unsigned char* p) {
        u32x4 f = *reinterpret_cast<const u32x4*>(p);
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t t = ((f[j] & 0x7fff7fffu) + T::kNonFinite) & 0x80008000u;
            f[j] &= ~((t >> 15) * 0xffffu);
            bad |= t;
        }
        if (bad) *reinterpret_cast<u32x4*>(p) = f;
        any = any || __builtin_amdgcn_ballot_w64(bad != 0);
    }
    // Every wave of the workgroup: whether any of them held something back. Uses LDS that no one reads
    // any more.
    __device__ __forceinline__ void share(unsigned char* lds) {
        __syncthreads();
        int* const flag = reinterpret_cast<int*>(lds);
        if ((threadIdx.x & 63) == 0) flag[threadIdx.x >> 6] = any;
        __syncthreads();
        any = (flag[0] | flag[1] | flag[2] | flag[3]) != 0;
        __syncthreads();
    }
    // Rows [r0, r0 + n), dims [d0, d0 + dims), which this wave has stored.
    template <typename SPAN>
    __device__ __forceinline__ void add(const CausalArgs& a, const CausalItem& it, const SPAN& span, int kvh, int r0, int n, int d0,
                                        int dims) const {
        __threadfence();
        const uint32_t g = uint32_t(a.group);
        for (int b = 0; b < span.blocks; b++) {
            if (!mixed(span.first(b), SPAN::kKeys)) continue;
            for (int key = span.first(b); key < span.end(b); key++) {
                const uint16_t* const v = span.template value_row<HD>(b, key, kvh);
                for (int d = d0 + int(threadIdx.x & 63); d < d0 + dims; d += 64) {
                    const uint16_t x = v[d];
                    if (((x & 0x7fffu) + (T::kNonFinite & 0xffffu)) < 0x8000u) continue;
                    for (int row = 0; row < n; row++) {
                        const uint32_t r = uint32_t(r0 + row);
                        const int i = int(r / g);
                        if (key > i + it.shift || (a.window && key <= i + it.shift - a.window)) continue;
                        if (it.part == kDirect) {
                            uint16_t* o = a.out + (size_t(it.q_token) + r / g) * size_t(a.out_stride) + (size_t(kvh) * g + r % g) * HD + d;
                            *o = uint16_t(T::pack(T::value(*o) + T::value(x), 0.0f));
                        } else {
                            a.part_o[(size_t(kvh) * a.part_rows + it.part + (r - it.row0)) * HD + d] += T::value(x);
                        }
                    }
                }
            }
        }
    }
};

// The waves that took different key blocks of the same rows join: all but the first leave their maximum, sum
// and accumulators in LDS, the first adds them in order. Every wave of the workgroup comes here; LDS is
// no longer read.
template <typename T, int HD, int DW, int KW>
struct JoinKeys {
    using W = Rows<T, HD, DW>;
    static constexpr int kAcc = W::DT * 16;
    static constexpr int kLds = (KW - 1) * DW * 64 * (kAcc + 2) * 4;
    static __device__ __forceinline__ void run(W& w, int kw, int dims, int lane, unsigned char* lds) {
        float* const j = reinterpret_cast<float*>(lds);
        if (kw > 0) {
            float* const p = j + (((kw - 1) * DW + dims) * (kAcc + 2)) * 64 + lane;
            p[0] = w.m;
            p[64] = w.l;
#pragma unroll
            for (int d = 0; d < W::DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) p[(2 + d * 16 + e) * 64] = w.o[d][e];
        }
        __syncthreads();
        if (kw > 0) return;
        float top = w.m;
#pragma unroll
        for (int k = 1; k < KW; k++) top = fmaxf(top, j[((k - 1) * DW + dims) * (kAcc + 2) * 64 + lane]);
        const float f0 = w.m == top ? 1.0f : __builtin_amdgcn_exp2f(w.m - top);
        w.l *= f0;
#pragma unroll
        for (int d = 0; d < W::DT; d++) w.o[d] *= f0;
        for (int k = 1; k < KW; k++) {
            const float* const p = j + ((k - 1) * DW + dims) * (kAcc + 2) * 64 + lane;
            const float mk = p[0], f = mk == top ? 1.0f : __builtin_amdgcn_exp2f(mk - top);
            w.l += p[64] * f;
#pragma unroll
            for (int d = 0; d < W::DT; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) w.o[d][e] += p[(2 + d * 16 + e) * 64] * f;
        }
        w.m = top;
    }
};

// Entry `at` of a list in memory, or of the one among the arguments, in scalar registers.
template <typename E>
__device__ __forceinline__ E uniform_entry(const E* list, const E* few, uint32_t at) {
    constexpr int N = sizeof(E) / 4;
    uint32_t w[N];
    if (list) {
        const uint32_t* const p = reinterpret_cast<const uint32_t*>(list + at);
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = uint32_t(__builtin_amdgcn_readfirstlane(int(p[i])));
    } else {
        const uint32_t* const p = reinterpret_cast<const uint32_t*>(few + at);
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = uint32_t(__builtin_amdgcn_readfirstlane(int(p[i])));
    }
    E e;
    __builtin_memcpy(&e, w, sizeof(E));
    return e;
}

}  // namespace
}  // namespace ge
