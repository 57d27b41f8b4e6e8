// The 8-bit form of an activation (mvs_act8_quantize): blocks of 32 values share one power of two 2^k.
//
//   k = the smallest integer >= -126 with round(max|x| / 2^k) <= 127;   q = round-to-nearest-even(x / 2^k), |q| <= 127
//
// A power of two makes the division exact: the codes depend on the values alone, not on how a quotient was rounded, and a code
// times 2^k is exact in float32 and bfloat16 (seven bits).  With max|x| = m 2^e, 1 <= m < 2: 64 m < 127.5 gives k = e - 6, else
// e - 5 -- the error of a value is at most half a step, 2^(k-1) <= max|x| / 127.
#pragma once
#include "mvs_common.h"

namespace mvs {

constexpr int kAct8Block = 32;
constexpr unsigned kAct8Nan = 255;      // scale byte of a block that holds an Inf or NaN

// amax_bits: the bits of max|x| (sign cleared: they order like the values, Inf and NaN above every number) -> scale byte k + 127
__device__ __forceinline__ unsigned act8_scale_byte(unsigned amax_bits) {
    if (amax_bits >= 0x7f800000u) return kAct8Nan;
    const int e = (int)(amax_bits >> 23) - 6 + ((amax_bits & 0x7fffffu) >= 0x7f0000u ? 1 : 0);
    return (unsigned)(e < 1 ? 1 : e);
}
// 2^-k and 2^k of a scale byte in 1 .. 250 (both normal numbers)
__device__ __forceinline__ float act8_inverse(unsigned byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float act8_step(unsigned byte) { return byte == kAct8Nan ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23); }
__device__ __forceinline__ int act8_code(float x, float inverse) { return (int)__builtin_rintf(x * inverse); }
__device__ __forceinline__ unsigned act8_pack4(int a, int b, int c, int d) {
    return (unsigned)(a & 255) | (unsigned)(b & 255) << 8 | (unsigned)(c & 255) << 16 | (unsigned)d << 24;
}
// code j of four packed ones
__device__ __forceinline__ float act8_value(unsigned packed, int j, float step) { return (float)((int)(packed << (24 - 8 * j)) >> 24) * step; }

__device__ __forceinline__ unsigned umax_xor(unsigned v, int lanes) {
    const unsigned o = (unsigned)__shfl_xor((int)v, lanes);
    return v > o ? v : o;
}

}  // namespace mvs
