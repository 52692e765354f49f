// Rows of 16-bit floats as whole numbers of 8 bits and a scale: the index keys and queries of the block selection.
//
// scale = max|x| / 127, code = x / scale rounded to 32 bits and then to a whole number, halves to even (0 where the scale
// is 0). The quotient is a division only where a product with the reciprocal could round to another whole number: product
// and quotient differ by at most 127 * (2^-22.9 + 2^-24) < 3e-5, so a product further than 4e-5 from a half has the
// quotient's whole number.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ekv {

__device__ __forceinline__ float code_scale(float most) { return most / 127.0f; }

// The codes of 8 elements of a row whose largest magnitude gives `scale`, the first in the first word's low byte. All
// lanes of a wave call it.
__device__ __forceinline__ void code_words(const float (&x)[8], float scale, uint32_t (&words)[2]) {
    const float divisor = scale > 0 ? scale : 1.0f, inverse = 1.0f / divisor;
    float code[8];
    // A reciprocal of a tiny scale may pass the largest number.
    bool close = divisor < 1e-30f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float product = x[j] * inverse;
        code[j] = rintf(product);
        close |= fabsf(product - code[j]) > 0.5f - 4e-5f;
    }
    if (__ballot(close) != 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            code[j] = rintf(x[j] / divisor);
        }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        words[w] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            words[w] |= (static_cast<uint32_t>(static_cast<int32_t>(code[4 * w + j])) & 0xffu) << (8 * j);
        }
    }
}

}  // namespace ekv
