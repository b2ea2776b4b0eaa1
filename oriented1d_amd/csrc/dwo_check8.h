// 8-bit checkpoints: what a backward pass needs of an activation, in one byte a value and one more for every 32 of them.
//
// Groups of 32 neighbours along a row share a power of two s = 2^(floor(log2(largest magnitude)) - 6), at least 2^-126, and hold
// q = round(x / s), ties to even, in [-127, 127].  The byte of a group is the biased exponent of s, so that it is a float's; 0: all values are
// zero, 255: one of them was not finite, and all come back as NaN, so that an overflow still shows in the gradients.  A power of two
// costs up to a bit against largest / 127, but q s is exact in bf16 and fp16: the products read what is held without another rounding.
#pragma once

#include "dwo_product.h"

namespace dwo {

constexpr int kGroup8 = 32;

__device__ __forceinline__ unsigned group_exponent(float most) {  // most: largest magnitude, NaN or infinite where one is
    const unsigned e = __float_as_uint(most) >> 23 & 0xff;
    return e == 0xff ? 255u : most == 0.f ? 0u : e > 7u ? e - 6u : 1u;
}
__device__ __forceinline__ float group_scale(unsigned e) { return __uint_as_float(e == 255u ? 0x7fc00000u : e << 23); }
// what a value is multiplied with on the way in: 1 / s, 0 where nothing is held
__device__ __forceinline__ float group_inverse(unsigned e) { return e == 0u || e == 255u ? 0.f : __uint_as_float((254u - e) << 23); }
__device__ __forceinline__ int quantum(float v, float inverse) {
    return (int)__builtin_amdgcn_fmed3f(__builtin_rintf(v * inverse), -127.f, 127.f);
}
// (a maximum of magnitudes as integers orders NaN above everything)
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

}  // namespace dwo
