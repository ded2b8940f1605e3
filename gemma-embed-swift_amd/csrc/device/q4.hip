// Products of few rows with 4-bit weights (gfx950): y[r][n] = sum_k x[r][k] w[n][k].
//
// The weights are read once; a pass over them is the floor. Each wave takes 16 weight rows (n) and up
// to 64 rows of x on v_mfma_f32_16x16x32: A = x, B = the weights' integers q of one group of 32 columns (a
// dword a lane). A group's products come out in fp32 and are added to the accumulators times the group's
// scale in fp32,
//   y += d (sum_k (q - 8) x)  [Q4_0],   y += d (sum_k q x) + m (sum_k x)  [Q4_1],
// so nothing is rounded but the fp32 sums. sum_k x is the same instruction with a constant B.
// A lane's accumulators are rows of x (4 (l / 16) + i) of one weight row (l % 16): one scale a lane and
// group. Row m of x stands at A's row 4 (m % 4) + m / 4, so that up to 4 rows fill the accumulators'
// first register only, 8 the first two, and the others are left out of the scaling.
// The waves of a workgroup take the column tiles in turn and join through LDS.
//
// Those steps leave fp32's range where the products w x need not: an infinite x as inf - inf between a product and
// the sum of x that corrects it, and bf16 x from 2^118 on times the integers, 31 times its size in 32 columns.
// A sum that comes out infinite or NaN is therefore taken again from the products themselves, in 64 bits.
#include "common.hpp"
#include "q4.hpp"

namespace ge {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// The integers of a dword as 8 values of x's type, plus kOffset: fp16 takes them exactly, as 1024 + q less
// 1024 or 1032; bf16, which has no packed addition, as 16 + q (0x4180 | q << 3), and the sum of x corrects
// for it. Converting them instead took 22.5 us for one row by 8192 x 8192 and 20.2 this way. (As fp16
// subnormals, the nibbles' bits as they are, they would need no arithmetic, but the matrix instruction keeps
// fewer bits of such products.)
struct F16 {
    template <bool MIN>
    static __device__ __forceinline__ u32x4 unpack(uint32_t w) {
        // 0x6400 | q is 1024 + q. The mask in a vector register lets one instruction mask and set.
        const half2_t base = {_Float16(MIN ? 1024 : 1032), _Float16(MIN ? 1024 : 1032)};
        uint32_t mask = 0x000f000fu;
        asm("" : "+v"(mask));
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t pair = ((w >> (4 * i)) & mask) | 0x64006400u;
            r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, pair) - base);
        }
        return r;
    }
    static __device__ __forceinline__ float4_t mfma(u32x4 a, u32x4 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float value(uint16_t x) { return h2f(x); }
    static constexpr float kOffset = 0.0f;
    static constexpr uint32_t kOnes = 0x3c003c00u, kMinus24 = 0;
};
struct BF16 {
    template <bool MIN>
    static __device__ __forceinline__ u32x4 unpack(uint32_t w) {
        uint32_t mask = 0x00780078u;
        asm("" : "+v"(mask));
        return u32x4{((w << 3) & mask) | 0x41804180u, ((w >> 1) & mask) | 0x41804180u, ((w >> 5) & mask) | 0x41804180u,
                     ((w >> 9) & mask) | 0x41804180u};
    }
    static __device__ __forceinline__ float4_t mfma(u32x4 a, u32x4 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float value(uint16_t x) { return __uint_as_float(uint32_t(x) << 16); }
    static constexpr float kOffset = 16.0f;
    static constexpr uint32_t kOnes = 0x3f803f80u, kMinus24 = 0xc1c0c1c0u;
};

__device__ __forceinline__ u32x4 splat(uint32_t x) { return u32x4{x, x, x, x}; }

// One lane a (row block, tile): every thread writes the dwords it owns, padding as zeros.
__global__ __launch_bounds__(64) void q4_repack_kernel(const unsigned char* __restrict__ blocks, const Q4Dev w) {
    const int lane = threadIdx.x, b = blockIdx.x / w.tiles, t = blockIdx.x % w.tiles;
    const int groups = w.cols / 32, bytes = w.m ? 20 : 18;
    const size_t tile = size_t(blockIdx.x);
    const int row = b * 16 + (lane & 15), e0 = 8 * (lane >> 4);
    u32x4 q = splat(0);
    for (int g = 0; g < 4; g++) {
        const int group = t * 4 + g;
        if (row < w.rows && group < groups) {
            const unsigned char* p = blocks + (size_t(row) * groups + group) * bytes + bytes - 16;
            uint32_t v = 0;
            for (int e = 0; e < 8; e++) {
                const int at = e0 + e;
                const uint32_t nibble = (p[at & 15] >> (at >= 16 ? 4 : 0)) & 15u;
                v |= nibble << (4 * (e & 1 ? 4 + e / 2 : e / 2));
            }
            q[g] = v;
        }
    }
    *reinterpret_cast<u32x4*>(w.q + tile * 256 + lane * 4) = q;
    // lane = 4 row + group
    const int r = b * 16 + (lane >> 2), group = t * 4 + (lane & 3);
    const bool in = r < w.rows && group < groups;
    const unsigned char* p = blocks + (size_t(r) * groups + group) * bytes;
    w.d[tile * 64 + lane] = in ? uint16_t(p[0] | p[1] << 8) : 0;
    if (w.m) w.m[tile * 64 + lane] = in ? uint16_t(p[2] | p[3] << 8) : 0;
}

template <Q4Out OUT>
__device__ __forceinline__ void store(void* y, size_t at, float v) {
    if (OUT == kQ4F32)
        static_cast<float*>(y)[at] = v;
    else if (OUT == kQ4F16)
        static_cast<_Float16*>(y)[at] = _Float16(v);
    else
        static_cast<__bf16*>(y)[at] = __bf16(v);
}

// sum_k x[k] w[n][k] of one row of x and one of the weights from its definition.
template <typename T, bool MIN>
__device__ __forceinline__ float product_again(const Q4Dev& w, const uint16_t* x, int n) {
    double sum = 0.0;
    for (int group = 0; group < w.cols / 32 && sum == sum; group++) {
        const size_t tile = size_t(n >> 4) * w.tiles + (group >> 2);
        const int at = (n & 15) * 4 + (group & 3);
        const double d = double(h2f(w.d[tile * 64 + at])), m = MIN ? double(h2f(w.m[tile * 64 + at])) : 0.0;
        for (int quad = 0; quad < 4; quad++) {
            const uint32_t q = w.q[tile * 256 + quad * 64 + at];
            for (int e = 0; e < 8; e++) {
                const int v = int((q >> (4 * (e & 1 ? 4 + e / 2 : e / 2))) & 15u) - (MIN ? 0 : 8);
                sum += (d * double(v) + m) * double(T::value(x[group * 32 + quad * 8 + e]));
            }
        }
    }
    return float(sum);
}

// What a wave reads of one column tile: its dwords of the weights, the scales (and minima) of its row's
// four groups, of BLOCKS weight blocks, and (unless x is in LDS) its fragments of x.
template <int NT, int BLOCKS, bool MIN, bool XLDS>
struct Tile {
    u32x4 q[BLOCKS], x[XLDS ? 1 : NT][4];
    u32x2 d[BLOCKS], m[BLOCKS];

    // block(k, tile): the matrix of block k, and the place of its tile.
    template <typename F>
    __device__ __forceinline__ void load(const Q4Args& a, F&& block, const uint16_t* const (&xr)[NT], int t, int lane) {
#pragma unroll
        for (int k = 0; k < BLOCKS; k++) {
            size_t tile;
            const Q4Dev& w = block(k, tile);
            q[k] = *reinterpret_cast<const u32x4*>(w.q + tile * 256 + lane * 4);
            d[k] = *reinterpret_cast<const u32x2*>(w.d + tile * 64 + (lane & 15) * 4);
            if (MIN) m[k] = *reinterpret_cast<const u32x2*>(w.m + tile * 64 + (lane & 15) * 4);
        }
        if (!XLDS) {
            // a group past the last column is read from the last one, and cleared before its use
#pragma unroll
            for (int g = 0; g < 4; g++)
#pragma unroll
                for (int j = 0; j < NT; j++)
                    x[j][g] = *reinterpret_cast<const u32x4*>(xr[j] + min(t * 128 + g * 32, a.w.cols - 32));
        }
    }
};

// Rows of x that are kept in LDS, whole, where they fit (kXBytes): a fragment read from memory moves 1 KB
// through the CU's address unit whatever the rows, 4 KB a tile beside 1.1 of weights.
constexpr int kXRows = 4, kXBytes = 64 << 10;

// Eight waves share the tiles of up to four rows (8192 x 8192: 20.1 us a call, 21.7 with four), four those of
// more (37 rows by 1001 x 2048 17.3 us, 18.5 with eight), whose registers leave room for fewer.
constexpr int kQ4Sums = 8;
template <bool XLDS>
constexpr int kQ4Waves = XLDS ? 8 : 4;

// NT: 16-row tiles of x; MR: accumulator registers in use (4 MR rows of a tile). RB: row blocks of a
// workgroup, which a fragment of x then serves. MATS: 1, or 2 for the GeGLU form. MIN: the weights have
// minima (Q4_1).
template <typename T, int NT, int MR, int RB, int MATS, bool MIN, bool XLDS, Q4Out OUT>
__global__ __launch_bounds__(512) void gemv_q4_kernel(const Q4Args a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char q4_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int waves = int(blockDim.x >> 6), quad = lane >> 4;
    const int tiles = a.w.tiles, cols = a.w.cols, last = (a.w.rows - 1) >> 4;
    constexpr int BLOCKS = RB * MATS;
    const int r0 = int(blockIdx.y) * (16 * NT);
    // the row of x at this lane's row of A; rows past the last one repeat it, and are not stored
    const int xrow = ((lane & 15) >> 2) + 4 * (lane & 3);
    const uint16_t* x[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) x[j] = a.x + size_t(min(r0 + 16 * j + xrow, a.rows - 1)) * cols + 8 * quad;
    // The tiles of this wave, AHEAD of them in flight (more gained nothing: other waves cover the reads).
    constexpr int AHEAD = NT == 1 ? 2 : 1;
    Tile<NT, BLOCKS, MIN, XLDS> s[AHEAD];
    auto load = [&](Tile<NT, BLOCKS, MIN, XLDS>& f, int t) {
        const int at = min(t, tiles - 1);
        // block k: row block k / MATS of the workgroup's (the last one again past the end), matrix k % MATS
        f.load(a, [&](int k, size_t& tile) -> const Q4Dev& {
            tile = size_t(min(int(blockIdx.x) * RB + k / MATS, last)) * tiles + at;
            return k % MATS ? a.up : a.w;
        }, x, at, lane);
    };
    // Every kernel adds up the same eight sums, of the tiles t = v mod 8, v = 0 .. 7, so a row's bits do not
    // depend on the rows beside it: eight waves take one each, four two, v and then v + 4.
    constexpr int SUMS = kQ4Sums / kQ4Waves<XLDS>;
    auto tiles_of = [&](int v) { return v < tiles ? (tiles - v + kQ4Sums - 1) / kQ4Sums : 0; };
    const int first = tiles_of(wave), count = first + (SUMS > 1 ? tiles_of(wave + kQ4Waves<XLDS>) : 0);
    auto tile_of = [&](int n) { return n < first ? wave + n * kQ4Sums : wave + kQ4Waves<XLDS> + (n - first) * kQ4Sums; };
#pragma unroll
    for (int i = 0; i < AHEAD; i++) load(s[i], tile_of(i));
    const unsigned char* xl = q4_lds;
    if (XLDS) {
        // 16-byte pieces, piece c of row r at (c rows + r)
        const int pieces = tiles * 16;
        for (int i = threadIdx.x; i < pieces * a.rows; i += blockDim.x) {
            const int r = i / pieces, c = i - r * pieces;
            *reinterpret_cast<u32x4*>(q4_lds + (size_t(c) * a.rows + r) * 16) =
                c * 8 < cols ? *reinterpret_cast<const u32x4*>(a.x + size_t(r) * cols + c * 8) : splat(0);
        }
        xl += (quad * a.rows + min(xrow, a.rows - 1)) * 16;
        __syncthreads();
    }
    float* const part = reinterpret_cast<float*>(q4_lds);
    float acc[BLOCKS][NT][MR] = {};
    auto leave = [&](int v) {  // sum v for the join
#pragma unroll
        for (int k = 0; k < BLOCKS; k++)
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < MR; e++) {
                    part[(((v * BLOCKS + k) * NT + j) * MR + e) * 64 + lane] = acc[k][j][e];
                    acc[k][j][e] = 0.0f;
                }
    };
    for (int n0 = 0; n0 < count; n0 += AHEAD)
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (n0 + i >= count) break;
            if (SUMS > 1 && n0 + i == first) leave(wave);
            const int t = tile_of(n0 + i);
            // The weights of columns past the end are zeros; x must be too, for an infinity or NaN in its place.
            if (!XLDS && t * 128 + 128 > cols) {
#pragma unroll
                for (int g = 1; g < 4; g++)
#pragma unroll
                    for (int j = 0; j < NT; j++)
                        if (t * 128 + g * 32 >= cols) s[i].x[XLDS ? 0 : j][g] = splat(0);
            }
#pragma unroll
            for (int g = 0; g < 4; g++) {
                // Q4_1: sum_k x; Q4_0 of 16 + q: -24 sum_k x, where the product starts
                constexpr bool kStart = !MIN && T::kOffset != 0.0f;
                u32x4 xf[NT];
                float4_t sums[NT] = {};
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    xf[j] = XLDS ? *reinterpret_cast<const u32x4*>(xl + (t * 16 + g * 4) * a.rows * 16) : s[i].x[XLDS ? 0 : j][g];
                    if (MIN || kStart) sums[j] = T::mfma(xf[j], splat(MIN ? T::kOnes : T::kMinus24), float4_t{});
                }
#pragma unroll
                for (int k = 0; k < BLOCKS; k++) {
                    const u32x4 wf = T::template unpack<MIN>(s[i].q[k][g]);
                    const half4_t d = __builtin_bit_cast(half4_t, s[i].d[k]), m = __builtin_bit_cast(half4_t, s[i].m[k]);
                    const float least = __builtin_fmaf(-T::kOffset, float(d[g]), float(m[g]));
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        const float4_t p = T::mfma(xf[j], wf, kStart ? sums[j] : float4_t{});
#pragma unroll
                        for (int e = 0; e < MR; e++) {
                            float& y = acc[k][j][e];
                            y = __builtin_fmaf(float(d[g]), p[e], y);
                            if (MIN) y = __builtin_fmaf(least, sums[j][e], y);
                        }
                    }
                }
            }
            load(s[i], tile_of(n0 + i + AHEAD));
        }
    // Join in the order of the sums; each wave finishes every waves-th tile of x rows.
    const int parts = min(tiles, kQ4Sums);
    if (parts > 1) {
        if (XLDS) __syncthreads();
        leave(SUMS > 1 && count > first ? wave + kQ4Waves<XLDS> : wave);
        __syncthreads();
    }
    uint32_t again = 0;  // this lane's results of which a sum is not finite
#pragma unroll
    for (int j = 0; j < RB * NT; j++) {
        if (j % waves != wave) continue;
        const int rb = j / NT, t = j % NT, n = (int(blockIdx.x) * RB + rb) * 16 + (lane & 15);
#pragma unroll
        for (int e = 0; e < MR; e++) {
            float sum[MATS];
#pragma unroll
            for (int k = 0; k < MATS; k++) {
                const int block = rb * MATS + k;
                sum[k] = acc[block][t][e];
                if (parts > 1) {
                    sum[k] = part[((block * NT + t) * MR + e) * 64 + lane];
                    for (int v = 1; v < parts; v++) sum[k] += part[(((v * BLOCKS + block) * NT + t) * MR + e) * 64 + lane];
                }
            }
            const float y = MATS == 2 ? gelu_tanh(sum[0]) * sum[MATS - 1] : sum[0];
            const int r = r0 + 16 * t + quad + 4 * e;
            if (r < a.rows && n < a.w.rows) {
                store<OUT>(a.y, size_t(r) * a.w.rows + n, y);
                if (!__builtin_isfinite(sum[0]) || (MATS == 2 && !__builtin_isfinite(sum[MATS - 1]))) again |= 1u << (j * MR + e);
            }
        }
    }
    static_assert(RB * NT * MR <= 32, "a bit a result");
    for (; again; again &= again - 1) {
        const int at = __builtin_ctz(again), j = at / MR, e = at % MR;
        const int n = (int(blockIdx.x) * RB + j / NT) * 16 + (lane & 15), r = r0 + 16 * (j % NT) + quad + 4 * e;
        const uint16_t* const row = a.x + size_t(r) * cols;
        float y = product_again<T, MIN>(a.w, row, n);
        if (MATS == 2) y = gelu_tanh(y) * product_again<T, MIN>(a.up, row, n);
        store<OUT>(a.y, size_t(r) * a.w.rows + n, y);
    }
}

template <typename T, int NT, int MR, int RB, int MATS, bool MIN, bool XLDS, Q4Out OUT>
hipError_t run(hipStream_t s, const Q4Args& a) {
    const int waves = a.w.tiles < kQ4Waves<XLDS> ? a.w.tiles : kQ4Waves<XLDS>, parts = a.w.tiles < kQ4Sums ? a.w.tiles : kQ4Sums;
    const uint32_t join = parts > 1 ? uint32_t(parts * RB * MATS * NT * MR) * 256u : 0;
    const uint32_t x = XLDS ? uint32_t(a.rows * a.w.tiles) * 256u : 0;
    const dim3 grid(uint32_t((q4_row_blocks(a.w.rows) + RB - 1) / RB), uint32_t((a.rows + 16 * NT - 1) / (16 * NT)));
    launch_kernel(gemv_q4_kernel<T, NT, MR, RB, MATS, MIN, XLDS, OUT>, grid, dim3(uint32_t(waves) * 64), join > x ? join : x, s, a);
    return hipGetLastError();
}
template <typename T, int NT, int MR, int RB, int MATS, bool MIN, bool XLDS>
hipError_t run_out(hipStream_t s, const Q4Args& a, Q4Out out) {
    return out == kQ4F32   ? run<T, NT, MR, RB, MATS, MIN, XLDS, kQ4F32>(s, a)
           : out == kQ4F16 ? run<T, NT, MR, RB, MATS, MIN, XLDS, kQ4F16>(s, a)
                           : run<T, NT, MR, RB, MATS, MIN, XLDS, kQ4BF16>(s, a);
}
template <typename T, int NT, int MR, int RB, bool XLDS>
hipError_t run_form(hipStream_t s, const Q4Args& a, bool geglu, Q4Out out) {
    // the GeGLU form's two matrices already share x
    constexpr int PAIR = RB > 1 ? RB / 2 : 1;
    if (a.w.m) return geglu ? run_out<T, NT, MR, PAIR, 2, true, XLDS>(s, a, out) : run_out<T, NT, MR, RB, 1, true, XLDS>(s, a, out);
    return geglu ? run_out<T, NT, MR, PAIR, 2, false, XLDS>(s, a, out) : run_out<T, NT, MR, RB, 1, false, XLDS>(s, a, out);
}
template <typename T>
hipError_t run_rows(hipStream_t s, const Q4Args& a, bool geglu, Q4Out out) {
    if (a.rows <= kXRows && int64_t(a.rows) * a.w.tiles * 256 <= kXBytes) return run_form<T, 1, 1, 1, true>(s, a, geglu, out);
    if (a.rows <= 8) return run_form<T, 1, 2, 1, false>(s, a, geglu, out);
    // As many rows of x and of the weights a workgroup as leave a workgroup for every CU: the weights are
    // read once for each 16 NT rows, x once for each 16 RB weight rows (8192 x 8192 a call: 16 rows 32.7 us
    // with RB 1, 27.0 with 2; 64 rows 75 and 48; 37 rows by 1001 x 2048 17.4 at NT 1, 25 at 4).
    const int blocks = q4_row_blocks(a.w.rows) * (geglu ? 2 : 1), t = (a.rows + 15) / 16;
    if (t == 1 || blocks * ((t + 1) / 2) < 256) {
        if (blocks * t >= 1024) return run_form<T, 1, 4, 4, false>(s, a, geglu, out);
        return blocks * t >= 512 ? run_form<T, 1, 4, 2, false>(s, a, geglu, out) : run_form<T, 1, 4, 1, false>(s, a, geglu, out);
    }
    if (t == 2 || blocks * ((t + 3) / 4) < 256)
        return blocks * ((t + 1) / 2) >= 512 ? run_form<T, 2, 4, 2, false>(s, a, geglu, out) : run_form<T, 2, 4, 1, false>(s, a, geglu, out);
    return blocks * ((t + 3) / 4) >= 512 ? run_form<T, 4, 4, 2, false>(s, a, geglu, out) : run_form<T, 4, 4, 1, false>(s, a, geglu, out);
}

}  // namespace

hipError_t launch_q4_repack(hipStream_t s, const unsigned char* blocks, const Q4Dev& w) {
    if (w.rows <= 0 || w.cols <= 0 || w.cols % 32 || w.rows > kQ4MaxWeightRows || w.cols > kQ4MaxCols || w.tiles != q4_tiles(w.cols)) return hipErrorInvalidValue;
    const uint64_t n = uint64_t(q4_row_blocks(w.rows)) * uint64_t(w.tiles);
    if (n >= (uint64_t(1) << 32) / 64) return hipErrorInvalidValue;
    launch_kernel(q4_repack_kernel, dim3(uint32_t(n)), dim3(64), 0, s, blocks, w);
    return hipGetLastError();
}

hipError_t launch_gemv_q4(hipStream_t s, const Q4Args& a, bool bf16, bool geglu, Q4Out out) {
    if (a.rows < 0 || a.rows > kQ4MaxRows || a.w.rows <= 0 || (geglu && (a.up.rows != a.w.rows || a.up.cols != a.w.cols || !a.up.m != !a.w.m)))
        return hipErrorInvalidValue;
    if (a.rows == 0) return hipSuccess;
    return bf16 ? run_rows<BF16>(s, a, geglu, out) : run_rows<F16>(s, a, geglu, out);
}

}  // namespace ge
