// The two 16-bit operand types of the kernels that take either.
#pragma once

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

}  // namespace
}  // namespace ge
