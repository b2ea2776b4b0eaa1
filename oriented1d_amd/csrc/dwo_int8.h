// Rows in 8-bit integers: a row with largest magnitude a stands as q a / 127, q = 127 v / a to the nearest whole number, ties to even, decided
// on the quotient itself and not on a rounded one.  So a code is the same whatever kernel makes it, on a value that lies next to the middle of
// two (half of the largest one does, in 16 bits one value in a few hundred).
#pragma once

#include "dwo_product.h"

namespace dwo {

typedef int mma_i4 __attribute__((ext_vector_type(4)));

struct i8_t {};
// Products of 8-bit integers in the place of 16-bit values: a "value" of the core is a pair of them, its sums are whole numbers in the sums'
// registers.  The bytes of a fragment lie as those of 16-bit values do, and both operands share them.
template <>
struct Mma<i8_t> {
    static constexpr short kOne = 0, kHalf = 0;  // (no sums over an operand)
    static __device__ __forceinline__ mma_f4 run(mma_s8 a, mma_s8 b, mma_f4 c) {
        return __builtin_bit_cast(mma_f4, __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(mma_i4, a), __builtin_bit_cast(mma_i4, b),
                                                                                __builtin_bit_cast(mma_i4, c), 0, 0, 0));
    }
};

// 2^-59 .. 2^61; zero is.  Of two such numbers the product over 127, 2^-125 or more, has all its bits, as products with whole numbers have then
__device__ __forceinline__ bool near_one(float v) {
    const unsigned e = __float_as_uint(v) >> 23 & 0xff;
    return e - 68u <= 119u || v == 0.f;
}
constexpr float kWholes = 12582912.f;  // 1.5 2^23: a sum with it is rounded to a whole number, ties to even, whose low byte is the sum's

// The codes of a row, as the low bytes of words.  Sixteen bits: t = 127 v is exact (18 bits at the most), and a quotient t / a that is no middle of
// two whole numbers is 8 of its last places away from one or more (|254 t' - (2k + 1) a'| >= 1 for the whole numbers t' and a' that they are, below
// 2^11 times a power of two).  q + (t - q a) / a has the quotient's own rounding: the remainder is exact, a middle comes out as itself.
// (Largest magnitudes far from 1: of v and a divided by a power of two.)
template <typename T>
struct RowCodes {
    float a, inverse;
    int e;
    __device__ __forceinline__ void init(float most) {  // most: finite, not negative
        e = near_one(most) ? 0 : __builtin_amdgcn_frexp_expf(most);
        a = most > 0.f ? __builtin_amdgcn_ldexpf(most, -e) : 1.f;
        inverse = 1.f / a;
    }
    __device__ __forceinline__ unsigned code(float v) const {
        const float t = v * 127.f, q = t * inverse;
        return __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q, a, t), inverse, q) + kWholes);
    }
    __device__ __forceinline__ void codes(float (&v)[8], unsigned (&w)[8]) const {
        if (__builtin_expect(e != 0, 0)) {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __builtin_amdgcn_ldexpf(v[i], -e);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = code(v[i]);
    }
};
// fp32: in 64 bits t = 127 v is exact, and a quotient that is no middle is 2^-33 away from one or more.  It is known to 2^-45; rounded to multiples of
// 2^-40 (those of a sum with 1.5 2^12) a middle is one again, and no other value becomes one.
template <>
struct RowCodes<float> {
    double inverse;
    __device__ __forceinline__ void init(float most) { inverse = most > 0.f ? 127.0 / (double)most : 0.0; }
    __device__ __forceinline__ void codes(float (&v)[8], unsigned (&w)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const double q = ((double)v[i] * inverse + 6144.0) - 6144.0;
            w[i] = __float_as_uint((float)__builtin_rint(q) + kWholes);
        }
    }
};
// the low bytes of four words
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}


// Eight values of a row: words as they lie in memory, zeros behind the row
template <typename T>
struct RowPiece {
    mma_u4 word[sizeof(T) / 2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; k++) word[k] = mma_u4{0u, 0u, 0u, 0u};
    }
    __device__ __forceinline__ void read(const T *row, int piece, int C, bool wide) {
        const int c = piece * 8;
        if (wide && c < C) {
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; k++) word[k] = reinterpret_cast<const mma_u4 *>(row + c)[k];
        } else {
            T v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = c + e < C ? row[c + e] : from_float<T>(0.f);
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; k++) word[k] = reinterpret_cast<const mma_u4 *>(v)[k];
        }
    }
};
// The largest magnitude of pieces, as its bits: integers, which order infinities and NaN above everything
template <typename T>
struct RowMost {
    typedef unsigned short two __attribute__((ext_vector_type(2)));
    unsigned m = 0;  // (of two 16-bit values side by side)
    __device__ __forceinline__ void meet(const RowPiece<T> &p) {
#pragma unroll
        for (int k = 0; k < (int)sizeof(T) / 2; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (sizeof(T) == 4) {
                    m = max(m, p.word[k][i] & 0x7fffffffu);
                } else {
                    const two v = __builtin_bit_cast(two, p.word[k][i] & 0x7fff7fffu);
                    m = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(two, m), v));
                }
            }
    }
    // over LANES neighbouring lanes, as fp32 (not finite: infinity or NaN)
    template <int LANES>
    __device__ __forceinline__ float join() const {
        unsigned v = sizeof(T) == 4 ? m : max(m & 0xffffu, m >> 16);
#pragma unroll
        for (int off = 1; off < (LANES < 64 ? LANES : 64); off <<= 1) v = max(v, (unsigned)__shfl_xor((int)v, off, 64));
        if constexpr (sizeof(T) == 4) return __uint_as_float(v);
        else return to_float(__builtin_bit_cast(T, (uint16_t)v));
    }
};
template <typename T>
__device__ __forceinline__ mma_u2 piece_codes(const RowCodes<T> &r, const RowPiece<T> &p) {
    float v[8];
    unsigned w[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = to_float(reinterpret_cast<const T *>(p.word)[e]);
    r.codes(v, w);
    return mma_u2{low_bytes(w[0], w[1], w[2], w[3]), low_bytes(w[4], w[5], w[6], w[7])};
}

}  // namespace dwo
