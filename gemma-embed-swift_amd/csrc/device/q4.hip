// Products of few rows with 4-bit weights (gfx950): y[r][n] = sum_k x[r][k] w[n][k].
//
// The weights are read once; a pass over them is the floor. Each wave takes 16 weight rows (n) and up
// to 64 rows of x on v_mfma_f32_16x16x32: A = the weights' integers q of one group of 32 columns (a dword
// a lane, exact in fp16 and bf16), B = x. A group's products come out in fp32 and are added to the
// accumulators times the group's scale in fp32,
//   y += d (sum_k (q - 8) x)  [Q4_0],   y += d (sum_k q x) + m (sum_k x)  [Q4_1],
// so nothing is rounded but the fp32 sums. sum_k x is the same instruction with A = 1, and bf16's -8 with
// A = -8. The waves of a workgroup take the column tiles in turn and join through LDS.
#include "common.hpp"
#include "q4.hpp"

namespace ge {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

// The integers of a dword as 8 values of x's type. BIAS: what is subtracted from them here.
struct F16 {
    template <int BIAS>
    static __device__ __forceinline__ u32x4 unpack(uint32_t w) {
        // 0x6400 | q is 1024 + q
        const half2_t base = {_Float16(1024 + BIAS), _Float16(1024 + BIAS)};
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t pair = ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u;
            r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, pair) - base);
        }
        return r;
    }
    static __device__ __forceinline__ float4_t mfma(u32x4 a, u32x4 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    }
    static constexpr int kBias = 8;
    static constexpr uint32_t kOnes = 0x3c003c00u, kMinus8 = 0xc800c800u;
};
struct BF16 {
    template <int BIAS>
    static __device__ __forceinline__ u32x4 unpack(uint32_t w) {
        const uint32_t even = w & 0x0f0f0f0fu, odd = (w >> 4) & 0x0f0f0f0fu;  // nibbles 0 2 4 6, 1 3 5 7
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // pair i: nibbles i and 4 + i, bytes i / 2 and 2 + i / 2 of the even or the odd ones
            const uint32_t b = (i & 1 ? odd : even) >> (8 * (i >> 1));
            r[i] = __builtin_bit_cast(uint32_t, bf16x2_t{__bf16(float(b & 0xffu)), __bf16(float((b >> 16) & 0xffu))});
        }
        return r;
    }
    static __device__ __forceinline__ float4_t mfma(u32x4 a, u32x4 b, float4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static constexpr int kBias = 0;
    static constexpr uint32_t kOnes = 0x3f803f80u, kMinus8 = 0xc100c100u;
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
    // lane = 16 quad + 4 group + row
    const int r = b * 16 + (lane >> 4) * 4 + (lane & 3), group = t * 4 + ((lane >> 2) & 3);
    const bool in = r < w.rows && group < groups;
    const unsigned char* p = blocks + (size_t(r) * groups + group) * bytes;
    w.d[tile * 64 + lane] = in ? uint16_t(p[0] | p[1] << 8) : 0;
    if (w.m) w.m[tile * 64 + lane] = in ? uint16_t(p[2] | p[3] << 8) : 0;
}

// fp16 scales of one group's four rows.
__device__ __forceinline__ float4_t scales(const uint16_t* p) {
    const half4_t h = *reinterpret_cast<const half4_t*>(p);
    return float4_t{float(h[0]), float(h[1]), float(h[2]), float(h[3])};
}

template <Q4Out OUT>
__device__ __forceinline__ void store4(void* y, size_t at, float4_t v, int n) {
    for (int i = 0; i < n; i++) {
        if (OUT == kQ4F32)
            static_cast<float*>(y)[at + i] = v[i];
        else if (OUT == kQ4F16)
            static_cast<_Float16*>(y)[at + i] = _Float16(v[i]);
        else
            static_cast<__bf16*>(y)[at + i] = __bf16(v[i]);
    }
}

// NT: 16-row tiles of x. MATS: 1, or 2 for the GeGLU form. MIN: the weights have minima (Q4_1).
template <typename T, int NT, int MATS, bool MIN, Q4Out OUT>
__global__ __launch_bounds__(512) void gemv_q4_kernel(const Q4Args a) {
    extern __shared__ __attribute__((aligned(16))) float q4_lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6));
    const int waves = int(blockDim.x >> 6), quad = lane >> 4;
    const int b = int(blockIdx.x), tiles = a.w.tiles, cols = a.w.cols;
    const int r0 = int(blockIdx.y) * (16 * NT);
    const uint16_t* x[NT];
#pragma unroll
    for (int j = 0; j < NT; j++) x[j] = a.x + size_t(min(r0 + 16 * j + (lane & 15), a.rows - 1)) * cols + 8 * quad;
    float4_t acc[MATS][NT] = {};
    for (int t = wave; t < tiles; t += waves) {
        const size_t tile = size_t(b) * tiles + t;
        u32x4 q[MATS];
#pragma unroll
        for (int k = 0; k < MATS; k++) q[k] = *reinterpret_cast<const u32x4*>((k ? a.up : a.w).q + tile * 256 + lane * 4);
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int col = t * 128 + g * 32;
            if (col >= cols) break;
            u32x4 xf[NT];
            float4_t sums[NT];
#pragma unroll
            for (int j = 0; j < NT; j++) {
                xf[j] = *reinterpret_cast<const u32x4*>(x[j] + col);
                // Q4_1: sum_k x; bf16 Q4_0: -8 sum_k x
                if (MIN || T::kBias == 0) sums[j] = T::mfma(splat(MIN ? T::kOnes : T::kMinus8), xf[j], float4_t{});
            }
#pragma unroll
            for (int k = 0; k < MATS; k++) {
                const Q4Dev& w = k ? a.up : a.w;
                const u32x4 wf = T::template unpack<MIN ? 0 : T::kBias>(q[k][g]);
                const size_t at = tile * 64 + quad * 16 + g * 4;
                const float4_t d = scales(w.d + at);
                const float4_t m = MIN ? scales(w.m + at) : float4_t{};
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const float4_t p = T::mfma(wf, xf[j], MIN || T::kBias ? float4_t{} : sums[j]);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        acc[k][j][i] = __builtin_fmaf(d[i], p[i], acc[k][j][i]);
                        if (MIN) acc[k][j][i] = __builtin_fmaf(m[i], sums[j][i], acc[k][j][i]);
                    }
                }
            }
        }
    }
    // Join in the order of the waves; each wave finishes every waves-th tile of x rows.
    float4_t* const part = reinterpret_cast<float4_t*>(q4_lds);
    if (waves > 1) {
#pragma unroll
        for (int k = 0; k < MATS; k++)
#pragma unroll
            for (int j = 0; j < NT; j++) part[((wave * MATS + k) * NT + j) * 64 + lane] = acc[k][j];
        __syncthreads();
    }
    const int n0 = b * 16 + quad * 4, n = min(4, a.w.rows - n0);
#pragma unroll
    for (int j = 0; j < NT; j++) {
        if (j % waves != wave) continue;
        const int r = r0 + 16 * j + (lane & 15);
        float4_t sum[MATS];
#pragma unroll
        for (int k = 0; k < MATS; k++) {
            sum[k] = acc[k][j];
            if (waves > 1) {
                sum[k] = part[(k * NT + j) * 64 + lane];
                for (int v = 1; v < waves; v++) sum[k] += part[((v * MATS + k) * NT + j) * 64 + lane];
            }
        }
        if (MATS == 2) {
#pragma unroll
            for (int i = 0; i < 4; i++) sum[0][i] = gelu_tanh(sum[0][i]) * sum[MATS - 1][i];
        }
        if (r < a.rows) store4<OUT>(a.y, size_t(r) * a.w.rows + n0, sum[0], n);
    }
}

template <typename T, int NT, int MATS, bool MIN, Q4Out OUT>
hipError_t run(hipStream_t s, const Q4Args& a) {
    const int waves = a.w.tiles < 8 ? a.w.tiles : 8;
    const uint32_t lds = waves > 1 ? uint32_t(waves * MATS * NT) * 1024u : 0;
    const dim3 grid(uint32_t(q4_row_blocks(a.w.rows)), uint32_t((a.rows + 16 * NT - 1) / (16 * NT)));
    launch_kernel(gemv_q4_kernel<T, NT, MATS, MIN, OUT>, grid, dim3(uint32_t(waves) * 64), lds, s, a);
    return hipGetLastError();
}
template <typename T, int NT, int MATS, bool MIN>
hipError_t run_out(hipStream_t s, const Q4Args& a, Q4Out out) {
    return out == kQ4F32 ? run<T, NT, MATS, MIN, kQ4F32>(s, a) : out == kQ4F16 ? run<T, NT, MATS, MIN, kQ4F16>(s, a) : run<T, NT, MATS, MIN, kQ4BF16>(s, a);
}
template <typename T, int NT>
hipError_t run_form(hipStream_t s, const Q4Args& a, bool geglu, Q4Out out) {
    if (a.w.m) return geglu ? run_out<T, NT, 2, true>(s, a, out) : run_out<T, NT, 1, true>(s, a, out);
    return geglu ? run_out<T, NT, 2, false>(s, a, out) : run_out<T, NT, 1, false>(s, a, out);
}
template <typename T>
hipError_t run_rows(hipStream_t s, const Q4Args& a, bool geglu, Q4Out out) {
    return a.rows <= 16 ? run_form<T, 1>(s, a, geglu, out) : a.rows <= 32 ? run_form<T, 2>(s, a, geglu, out) : run_form<T, 4>(s, a, geglu, out);
}

}  // namespace

hipError_t launch_q4_repack(hipStream_t s, const unsigned char* blocks, const Q4Dev& w) {
    if (w.rows <= 0 || w.cols <= 0 || w.cols % 32 || w.tiles != q4_tiles(w.cols)) return hipErrorInvalidValue;
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
