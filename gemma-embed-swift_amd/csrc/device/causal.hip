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
#include "causal.hpp"
#include "common.hpp"

namespace ge {
namespace {

typedef short short4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// The two input types: the matrix instruction, two floats rounded to nearest even and packed, the power of
// two by which P is taken higher, and the bits whose sum with a value's magnitude reaches its sign bit iff
// its exponent is all ones.
struct F16 {
    static __device__ __forceinline__ float16_t mfma(u32x4 a, u32x4 b, float16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        return __builtin_bit_cast(uint32_t, half2_t{_Float16(x), _Float16(y)});
    }
    // sum + the packed pair's two values
    static __device__ __forceinline__ float add(uint32_t pair, float sum) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, pair), half2_t{_Float16(1), _Float16(1)}, sum, false);
    }
    static __device__ __forceinline__ float value(uint16_t x) { return h2f(x); }
    static constexpr float kRaise = 6.0f;
    static constexpr uint32_t kNonFinite = 0x04000400u;
};
struct BF16 {
    static __device__ __forceinline__ float16_t mfma(u32x4 a, u32x4 b, float16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        return __builtin_bit_cast(uint32_t, bf16x2_t{__bf16(x), __bf16(y)});
    }
    static __device__ __forceinline__ float add(uint32_t pair, float sum) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pair), bf16x2_t{__bf16(1.0f), __bf16(1.0f)}, sum, false);
    }
    static __device__ __forceinline__ float value(uint16_t x) { return __uint_as_float(uint32_t(x) << 16); }
    static constexpr float kRaise = -32.0f;
    static constexpr uint32_t kNonFinite = 0x00800080u;
};

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
    // as the source's, so that a wave's chunks of a row group share one offset register.
    template <int PANEL>
    static __device__ __forceinline__ void copy(__amdgpu_buffer_rsrc_t r, unsigned char* block, int k8, uint32_t off) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            r, (__attribute__((address_space(3))) void*)(block + (PANEL * (BK / 8) + k8) * 1024 - PANEL * 128), 16, off, 0, PANEL * 128, 0);
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

// The key blocks of an item: those of its prefix keys, then those of its own, none of both.
template <int BK>
struct Span {
    int own0, blocks;      // the first block of own keys, all blocks
    int lo, end0, skip;    // the item's first key, the end of its prefix keys, the keys that block own0 - 1 lacks
    int hi;
    uint32_t own_row;      // + key: its row of k and v, modulo 2^32

    __device__ __forceinline__ Span(const CausalArgs& a, const CausalItem& it) : lo(int(it.k_lo)), hi(int(it.k_hi)) {
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
};

// Fragments read ahead of their products (four spill at head dim 256).
template <int HD>
constexpr int kFragmentsAhead = HD == 256 ? 3 : 4;

// 32 rows of one KV head: queries in registers, accumulators, running maximum and sum. DW waves can hold
// the same rows: they all compute the scores and each takes its share of the head's dims in the product.
template <typename T, int HD, int DW>
struct Rows {
    static constexpr int KS = HD / 16, DT = HD / 32 / DW;
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
        const uint16_t* p = a.q + (size_t(it.q_token) + i) * size_t(a.q_stride) + size_t(head) * HD + (lane >> 5) * 8;
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

        __device__ __forceinline__ void scores(const Rows& w, const unsigned char* K, int lane) {
            const int key = lane & 31, f = (key >> 1) & 7;
            const unsigned char* at[4];
#pragma unroll
            for (int c = 0; c < 4; c++) at[c] = K + key * 128 + (((2 * c + (lane >> 5)) ^ f) * 16);
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
                s[t] = T::mfma(ring[i % kAhead], w.q[k], s[t]);
                if (i + kAhead < KT * KS) read(i + kAhead);
            }
        }

        __device__ __forceinline__ bool sees_all(const Rows& w, int kb, int end) const {
            return kb + BK <= end && kb + BK - 1 <= w.hi_all && kb >= w.lo_all;
        }

        // Hidden keys and those from `end` on to -inf, the running maximum, and P.
        __device__ __forceinline__ void softmax(Rows& w, int kb, int end, float c, int lane, u32x4 (&p)[2 * KT]) {
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
// of which some of the item's rows see a key that others do not can hold such a key. Their V is cleared of
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
        return (kb + bk - 1 > hi_all && hi_all < hi_any) || (kb < lo_all && lo_any < lo_all);
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
    template <int BK>
    __device__ __forceinline__ void add(const CausalArgs& a, const CausalItem& it, const Span<BK>& span, int kvh, int r0, int n, int d0,
                                        int dims) const {
        __threadfence();
        const uint32_t g = uint32_t(a.group);
        for (int b = 0; b < span.blocks; b++) {
            if (!mixed(span.first(b), BK)) continue;
            for (int key = span.first(b); key < span.end(b); key++) {
                const uint16_t* const v = (b < span.own0 ? a.prefix_v + size_t(key) * size_t(a.v_stride)
                                                         : a.v + (size_t(it.key0) + size_t(key - a.prefix_len)) * size_t(a.v_stride)) +
                                          size_t(kvh) * HD;
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
        // a part that saw no key has nothing to add, whatever its rows hold
        const float f = ml.y == 0.0f ? 0.0f : ml.x == top ? 1.0f : __builtin_amdgcn_exp2f(ml.x - top);
        sum += ml.y == 0.0f ? 0.0f : ml.y * f;
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
                const bool none = i0 + i >= n || __shfl(ml.y, k, 64) == 0.0f;
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
