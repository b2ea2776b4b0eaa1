// Rows in 8-bit integers: a row with largest magnitude a stands as q a / 127, q = 127 v / a to the nearest whole number, ties to even, decided
// on the quotient itself and not on a rounded one.  So a code is the same whatever kernel makes it, on a value that lies next to the middle of
// two (half of the largest one does, in 16 bits one value in a few hundred).
#pragma once

#include "dwo_product.h"

namespace dwo {

struct i8_t {};
// Products of 8-bit integers in the place of 16-bit values: a "value" of the core is a pair of them, its sums are whole numbers in the sums'
// registers.  The bytes of a fragment lie as those of 16-bit values do, and both operands share them.
template <>
struct Mma<i8_t> {
    static constexpr short kOne = 0, kHalf = 0;  // (no sums over an operand)
    static __device__ __forceinline__ mma_f4 run(mma_s8 a, mma_s8 b, mma_f4 c) {
        typedef int i4 __attribute__((ext_vector_type(4)));
        return __builtin_bit_cast(mma_f4, __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4, a), __builtin_bit_cast(i4, b), __builtin_bit_cast(i4, c), 0, 0, 0));
    }
};

// The codes of a row.  Sixteen bits: w = v / 2^e and t = 127 w are exact (18 bits at the most), and a quotient that is no middle of two whole
// numbers is 8 of its last places away from one or more (|254 t' - (2k + 1) a'| >= 1 for the whole numbers t' and a' that they are, below 2^11 times
// a power of two).  q0 + (t - q0 m) / m has the quotient's own rounding: the remainder is exact, a middle comes out as itself.
template <typename T>
struct RowCodes {
    float m, inverse;
    int e;
    __device__ __forceinline__ void init(float most) {  // most: finite, not negative
        const bool some = most > 0.f;
        e = some ? __builtin_amdgcn_frexp_expf(most) : 0;
        m = some ? __builtin_amdgcn_frexp_mantf(most) : 1.f;
        inverse = 1.f / m;
    }
    __device__ __forceinline__ int code(float v) const {
        const float t = __builtin_amdgcn_ldexpf(v, -e) * 127.f;
        const float q = t * inverse;
        return (int)__builtin_rintf(__builtin_fmaf(__builtin_fmaf(-q, m, t), inverse, q));
    }
};
// fp32: in 64 bits t = 127 v is exact, and a quotient that is no middle is 2^-33 away from one or more.  It is known to 2^-45; rounded to multiples of
// 2^-40 (those of a sum with 1.5 2^12) a middle is one again, and no other value becomes one.
template <>
struct RowCodes<float> {
    double inverse;
    __device__ __forceinline__ void init(float most) { inverse = most > 0.f ? 127.0 / (double)most : 0.0; }
    __device__ __forceinline__ int code(float v) const {
        const double q = ((double)v * inverse + 6144.0) - 6144.0;
        return (int)__builtin_rint(q);
    }
};
// (a maximum of magnitudes as integers orders infinities and NaN above everything)
__device__ __forceinline__ bool finite_bits(unsigned most) { return most < 0x7f800000u; }

}  // namespace dwo
