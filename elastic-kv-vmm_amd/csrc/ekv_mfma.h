// Matrix instructions and conversions of the attention kernels, for both 16-bit types.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ekv {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t words4 __attribute__((ext_vector_type(4)));   // 8 elements
typedef uint32_t words2 __attribute__((ext_vector_type(2)));   // 4 elements

struct Bf16 {
    typedef __bf16 x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 x2 __attribute__((ext_vector_type(2)));
    // The weights exp(s - m) lie in [0, 2^kSlack]; bfloat16 has the exponents for them.
    static constexpr float kShift = 0.0f;
    static constexpr uint32_t kExponent = 0x7f807f80u;   // both halves' exponent bits
    static __device__ __forceinline__ f32x4 mfma16(words4 a, words4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(words4 a, words4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float low, float high) {
        return __builtin_bit_cast(uint32_t, x2{static_cast<__bf16>(low), static_cast<__bf16>(high)});
    }
    // The element in the word's low half if it is an infinity or a NaN, else 0.
    static __device__ __forceinline__ float unbounded(uint32_t word) {
        return (word & 0x7f80u) == 0x7f80u ? __uint_as_float(word << 16) : 0.0f;
    }
};

struct F16 {
    typedef _Float16 x8 __attribute__((ext_vector_type(8)));
    typedef _Float16 x2 __attribute__((ext_vector_type(2)));
    // Weights are kept as 2^7 exp(s - m): with kSlack at most 2^15, below the type's largest 65504, and small weights keep
    // their 11 bits down to 2^-21 of the reference instead of 2^-14. The sum carries the same factor, so it leaves the
    // quotient.
    static constexpr float kShift = 7.0f;
    static constexpr uint32_t kExponent = 0x7c007c00u;
    static __device__ __forceinline__ f32x4 mfma16(words4 a, words4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(words4 a, words4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float low, float high) {
        return __builtin_bit_cast(uint32_t, x2{static_cast<_Float16>(low), static_cast<_Float16>(high)});
    }
    static __device__ __forceinline__ float unbounded(uint32_t word) {
        return (word & 0x7c00u) == 0x7c00u
                   ? static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(word)))
                   : 0.0f;
    }
};

// 4 x 16 elements of a row-major LDS tile, transposed: each 16 lanes name four rows' 8-byte pieces (lane i the i % 4-th
// of row i / 4), and lane i gets column i of the four rows.
__device__ __forceinline__ words2 read_transposed(const char* at) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* lds;
    return __builtin_bit_cast(words2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(at)));
}

// Whether any half of the word is an infinity or a NaN.
template <typename T>
__device__ __forceinline__ bool not_finite(uint32_t word) {
    constexpr uint32_t kLow = T::kExponent & 0xffffu, kHigh = T::kExponent & 0xffff0000u;
    return (word & kLow) == kLow || (word & kHigh) == kHigh;
}

// The word with infinities and NaN replaced by 0.
template <typename T>
__device__ __forceinline__ uint32_t bounded(uint32_t word) {
    constexpr uint32_t kLow = T::kExponent & 0xffffu, kHigh = T::kExponent & 0xffff0000u;
    return word & ((word & kLow) == kLow ? 0xffff0000u : 0xffffffffu) & ((word & kHigh) == kHigh ? 0xffffu : 0xffffffffu);
}

}  // namespace ekv
