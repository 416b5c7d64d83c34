// Block-scaled 8-bit values: e4m3 (four exponent bits, three of mantissa, no infinities, largest 448) with one float32
// scale for 128 neighbours along K, a value being q * scale.
//
//   scale = max(amax / 448, 2^-126)     amax: the block's largest magnitude; the floor keeps 1 / scale finite and makes
//                                       a block of zeros (or of numbers too small for it) zeros with a normal scale
//   q     = round_to_e4m3(x * (1 / scale))
//
// amax / 448 is formed as amax * (1 / 448) and the quotient as a product with the rounded reciprocal: two float32
// roundings each, 2^-22 together, before one to 2^-4.  The largest element may come out as 448 (1 + 2^-22), which rounds
// to 448.  A NaN or an infinity makes its whole block NaN: amax is taken over the bits (NaN > infinity > every number), so
// the scale is NaN or infinite and every product with it is NaN.
#pragma once

#include "common.cuh"

namespace fp8 {

constexpr int BLOCK = 128;                            // elements along K (and, for weights, rows) that share a scale
constexpr float INV_MAX = 1.0f / 448.0f;
constexpr float MIN_SCALE = 1.17549435082228751e-38f;  // 2^-126

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
    const float s = __uint_as_float(amax_bits) * INV_MAX;
    return s < MIN_SCALE ? MIN_SCALE : s;             // NaN stays
}

// Four values as four bytes, the first in the lowest
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

}  // namespace fp8
