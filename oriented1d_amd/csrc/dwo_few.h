// Products of few rows, as one token or image makes them:  D[m][n] = sum_k x[m][k] w[n][k],  rows of both as they lie in memory.
//
// Bound by reading w once.  Tiles would fill sixteen rows or more with zeros and take w through LDS; here a wave has a column (gated: a
// gate and what it multiplies), its lanes sixteen bytes of w at a time straight to registers, and multiplies them with every row in
// fp32.  Where columns are few, two or four waves share one's sum; where they are many and rows three or more, a wave has two.
#pragma once

#include "dwo_act.h"

namespace dwo {

// Sixteen waves a CU: their loads in flight keep its memory busy.  Below it waves share columns (gated block 1024 -> 4096 -> 1024 in bf16, one row
// 7.0 us, without 8.3; four rows 11.2, 18.2), from it on two columns go to a wave from three rows on, whose pieces are then read for both
// (4096 -> 16384 -> 4096, four rows 101 us, 119 with one; 96 -> 256 -> 96 8.2, 6.2).
constexpr int kFewWaves = 4096;

// sixteen bytes of a row of w times as many values of x: pairs of 16-bit values by the instruction that adds two products to a sum in fp32
template <int N>
struct FewPiece {
    mma_u4 v[N];
};
template <typename T>
__device__ __forceinline__ float few_dot(const mma_u4 &a, const FewPiece<sizeof(float) / sizeof(T)> &x, float sum, T, float) {
    const T *w = reinterpret_cast<const T *>(&a);
#pragma unroll
    for (int e = 0; e < 16 / (int)sizeof(T); e++) sum = __builtin_fmaf(to_float(w[e]), __uint_as_float(x.v[e / 4][e % 4]), sum);
    return sum;
}
__device__ __forceinline__ float few_dot(const mma_u4 &a, const FewPiece<1> &x, float sum, bf16_t, bf16_t) {
    typedef __bf16 two __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; e++) sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(two, (unsigned)a[e]), __builtin_bit_cast(two, (unsigned)x.v[0][e]), sum, false);
    return sum;
}
__device__ __forceinline__ float few_dot(const mma_u4 &a, const FewPiece<1> &x, float sum, f16_t, f16_t) {
    typedef _Float16 two __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; e++) sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(two, (unsigned)a[e]), __builtin_bit_cast(two, (unsigned)x.v[0][e]), sum, false);
    return sum;
}
template <int CTRL>
__device__ __forceinline__ float few_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// over a wave, in every lane
__device__ __forceinline__ float few_total(float v) {
    v = few_add<0xB1>(v);   // quad_perm [1,0,3,2]
    v = few_add<0x4E>(v);   // quad_perm [2,3,0,1]
    v = few_add<0x141>(v);  // row_half_mirror
    v = few_add<0x140>(v);  // row_mirror
    const unsigned u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned w = __float_as_uint(__uint_as_float(s[0]) + __uint_as_float(s[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

struct FewPlain {
    static constexpr int kCols = 1;
    Values bias;
    Out out;
    __device__ __forceinline__ void operator()(long m, long n, const float (&v)[1]) const {
        out_one(out, m, n, v[0] + (bias.p != nullptr ? bias.at(n) : 0.f));
    }
};
struct FewGlu {
    static constexpr int kCols = 2;
    Values bias;  // [2 H]
    long rows, H, Hp;
    int act;
    float *keep;  // g, then u, [rows][Hp] each; or null
    float *h;  // [rows][H]
    __device__ __forceinline__ void operator()(long m, long n, const float (&v)[2]) const {
        const float g = v[0] + (bias.p != nullptr ? bias.at(n) : 0.f), u = v[1] + (bias.p != nullptr ? bias.at(H + n) : 0.f);
        if (keep != nullptr) keep[m * Hp + n] = g, keep[(rows + m) * Hp + n] = u;
        h[m * H + n] = act_value(act, g) * u;
    }
};

// U columns per wave.  along: waves that share them, 1, 2 or 4.  K in whole pieces of sixteen bytes.
template <typename TX, typename T, int R, int U, class End>
__global__ __launch_bounds__(256) void few_kernel(const TX *__restrict__ x, const T *__restrict__ w, long K, long N, long gap, int rows,
                                                  int along, End end) {
    constexpr int V = 16 / (int)sizeof(T), COLS = End::kCols;
    __shared__ float part[4][COLS][U * R];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = wave & ~(along - 1);
    const long n0 = ((long)blockIdx.x * 4 + wave) / along * U;
    float sum[U][COLS][R] = {};
#pragma unroll R > 2 ? 2 : 4
    for (long k = ((wave - first) * 64 + lane) * V; k < K; k += along * 64 * V) {
        mma_u4 a[U][COLS];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int c = 0; c < COLS; c++)
                a[u][c] = *reinterpret_cast<const mma_u4 *>(w + ((n0 + u < N ? n0 + u : N - 1) + c * gap) * K + k);
#pragma unroll
        for (int m = 0; m < R; m++) {
            const auto b = *reinterpret_cast<const FewPiece<sizeof(TX) / sizeof(T)> *>(x + (m < rows ? m : rows - 1) * K + k);
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int c = 0; c < COLS; c++) sum[u][c][m] = few_dot(a[u][c], b, sum[u][c][m], T{}, TX{});
        }
    }
    float mine[COLS] = {};  // lane u R + m: of column u and row m
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int c = 0; c < COLS; c++)
#pragma unroll
            for (int m = 0; m < R; m++) {
                const float v = few_total(sum[u][c][m]);
                mine[c] = lane == u * R + m ? v : mine[c];
            }
    if (along > 1) {
        if (lane < U * R)
#pragma unroll
            for (int c = 0; c < COLS; c++) part[wave][c][lane] = mine[c];
        __syncthreads();
        if (wave == first && lane < U * R)
#pragma unroll
            for (int c = 0; c < COLS; c++)
                for (int s = 1; s < along; s++) mine[c] += part[wave + s][c][lane];
    }
    const int m = lane % R;
    const long n = n0 + lane / R;
    if (wave == first && lane < U * R && m < rows && n < N) end(m, n, mine);
}

template <typename TX, typename T, class End>
int launch_few_typed(const void *x, const void *w, long K, long N, long gap, int rows, const End &end, hipStream_t st) {
    const bool two = rows > 2 && N >= kFewWaves;
    const long piece = 64 * 16 / (long)sizeof(T), units = two ? (N + 1) / 2 : N;
    int along = 1;
    while (along < 4 && units * along < kFewWaves && K >= 2 * along * piece) along *= 2;
    const dim3 grid((unsigned)((units * along + 3) / 4)), block(256);
    auto *kernel = rows == 1   ? few_kernel<TX, T, 1, 1, End>
                   : rows == 2 ? few_kernel<TX, T, 2, 1, End>
                   : two       ? few_kernel<TX, T, 4, 2, End>
                               : few_kernel<TX, T, 4, 1, End>;
    if constexpr (sizeof(T) == 4)
        if (rows > 4) kernel = two ? few_kernel<TX, T, 8, 2, End> : few_kernel<TX, T, 8, 1, End>;
    kernel<<<grid, block, 0, st>>>((const TX *)x, (const T *)w, K, N, gap, rows, along, end);
    return status();
}
// FLOAT: x in fp32 whatever w is
template <bool FLOAT, class End>
int launch_few(const void *x, const void *w, long K, long N, long gap, long rows, int dtype, const End &end, hipStream_t st) {
    switch (dtype) {
        case DWO_F32: return launch_few_typed<float, float>(x, w, K, N, gap, (int)rows, end, st);
        case DWO_BF16: return launch_few_typed<std::conditional_t<FLOAT, float, bf16_t>, bf16_t>(x, w, K, N, gap, (int)rows, end, st);
        default: return launch_few_typed<std::conditional_t<FLOAT, float, f16_t>, f16_t>(x, w, K, N, gap, (int)rows, end, st);
    }
}
// Up to eight rows in fp32, whose tiles take three planes made by another launch (gated block 1024 -> 4096 -> 1024: 13 us for one row and 25 for
// eight, as tiles 58 and 60; 4096 -> 16384 -> 4096: 141 and 220, 844 and 841), up to four in 16 bits (the first one 7.0 us for one row and 11.0 for
// four, as tiles 15.8 and 15.9; the second, of 403 MB, 72 and 96, 110 and 112; eight rows 15.8 and 123, 15.8 and 111; the slowest there
// is a layer of 4096 -> 32768 at four rows, 46 and 41).  For one row that is 3.6 TB/s of the first block's weights and 5.6 of the second's.
inline bool few(long rows, long K, int dtype) {
    return rows <= (dtype == DWO_F32 ? 8 : 4) && K % (dtype == DWO_F32 ? 4 : 8) == 0;
}

}  // namespace dwo
