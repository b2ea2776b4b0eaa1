// Linear layers at inference as products of 8-bit integers:
//   q = round(127 x / a), a the row's largest magnitude;  y = act((sum_c q_c p_c) (a / 127) s + b) for weights held as codes p and steps s.
//
// Whole numbers are summed, below 2^30 for 65536 channels: sums are exact and in any order, so that a row comes out the same whichever way it goes:
//   few rows, some, and many short ones: a kernel that takes its rows to codes on their way into LDS (int8_few_kernel, int8_resident_kernel);
//   others: a pass over x that leaves its codes and every row's a, and a product in tiles (dwo_product.h), whose epilogue does the rest.
// The tiles run at about the rate of the 16-bit products in operations a second times two; a product of short sums is bound by its results on their way out,
// which the 18 us of 77 MB are not hidden behind, and by the activation's 16 instructions a value.
#include <algorithm>

#include "dwo_act.h"
#include "dwo_int8.h"

namespace dwo {

constexpr int kCodePiece = 16;  // rows of codes are filled up to whole sixteen bytes
static long code_pitch(long C) { return (C + kCodePiece - 1) / kCodePiece * kCodePiece; }

// Codes of rows, LANES of a workgroup's threads a row, U pieces a lane (0: any number, read twice).  steps: a / 127 of each row or, for the product
// that follows, a itself; NaN where a value of the row is not finite, its codes are then zero.
template <typename T, int LANES, int U>
__global__ __launch_bounds__(256) void rows8_kernel(const T *__restrict__ x, int8_t *__restrict__ codes, float *__restrict__ steps, long rows,
                                                    int C, long pitch, bool raw) {
    __shared__ unsigned part[4];
    constexpr int ROWS = 256 / LANES;
    const int lane = threadIdx.x % LANES, pieces = (int)(pitch / 8);
    const bool wide = C % 8 == 0;
    for (long first = (long)blockIdx.x * ROWS; first < rows; first += (long)gridDim.x * ROWS) {
        const long row = first + threadIdx.x / LANES;
        const bool real = row < rows;
        const T *const at = x + (real ? row : first) * C;
        RowMost<T> largest;
        RowPiece<T> v[U > 0 ? U : 1];
        if constexpr (U > 0) {
#pragma unroll
            for (int u = 0; u < U; u++) v[u].clear();
#pragma unroll
            for (int u = 0; u < U; u++)
                if (lane + u * LANES < pieces) v[u].read(at, lane + u * LANES, C, wide);
#pragma unroll
            for (int u = 0; u < U; u++) largest.meet(v[u]);
        } else {
            for (int p = lane; p < pieces; p += LANES) v[0].read(at, p, C, wide), largest.meet(v[0]);
        }
        float a = largest.template join<LANES>();
        if constexpr (LANES > 64) {
            __syncthreads();
            if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = __float_as_uint(a);
            __syncthreads();
            a = __uint_as_float(max(max(part[0], part[1]), max(part[2], part[3])));
        }
        if (!real) continue;  // (with LANES above 64 all are)
        const bool finite = a < INFINITY;
        RowCodes<T> r;
        r.init(finite ? a : 0.f);
        if (lane == 0) steps[row] = !finite ? NAN : raw ? a : a / 127.f;
        mma_u2 *const to = reinterpret_cast<mma_u2 *>(codes + row * pitch);
        const mma_u2 none = mma_u2{0u, 0u};
        if constexpr (U > 0) {
#pragma unroll
            for (int u = 0; u < U; u++)
                if (lane + u * LANES < pieces) to[lane + u * LANES] = finite ? piece_codes(r, v[u]) : none;
        } else {
            for (int p = lane; p < pieces; p += LANES) v[0].read(at, p, C, wide), to[p] = finite ? piece_codes(r, v[0]) : none;
        }
    }
}

template <typename T>
static int launch_rows8(const void *x, int8_t *codes, float *steps, long rows, int C, bool raw, hipStream_t st) {
    const long pitch = code_pitch(C), pieces = pitch / 8;
    auto go = [&](auto *kernel, int lanes) {
        const long per = 256 / lanes, blocks = (rows + per - 1) / per;
        kernel<<<dim3((unsigned)(blocks < 1L << 20 ? blocks : 1L << 20)), dim3(256), 0, st>>>((const T *)x, codes, steps, rows, C, pitch, raw);
    };
    if (pieces <= 16) go(rows8_kernel<T, 16, 1>, 16);
    else if (pieces <= 64) go(rows8_kernel<T, 32, 2>, 32);
    else if (pieces <= 128) go(rows8_kernel<T, 64, 2>, 64);
    else if (pieces <= 256) go(rows8_kernel<T, 64, 4>, 64);
    else if (pieces <= 512) go(rows8_kernel<T, 64, 8>, 64);
    else if (pieces <= 1024) go(rows8_kernel<T, 256, 4>, 256);
    else go(rows8_kernel<T, 256, 0>, 256);
    return status();
}
static int rows8(const void *x, int8_t *codes, float *steps, long rows, int C, int dtype, bool raw, hipStream_t st) {
    if (dtype == DWO_F32) return launch_rows8<float>(x, codes, steps, rows, C, raw, st);
    if (dtype == DWO_BF16) return launch_rows8<bf16_t>(x, codes, steps, rows, C, raw, st);
    return launch_rows8<f16_t>(x, codes, steps, rows, C, raw, st);
}

constexpr float kInverse127 = 1.f / 127.f;
// What a whole number stands for: sum * (a / 127 * s).  Where a and s are not near 1, their product may be no number of fp32 though the
// result is one: then of their mantissas, and the power of two at the end, which gives the same bits where both do.
__device__ __forceinline__ float step_value(int sum, float a, float s) { return (float)sum * (a * kInverse127 * s); }
__device__ __forceinline__ float step_value_of_any(int sum, float a, float s) {
    return __builtin_amdgcn_ldexpf((float)sum * (__builtin_amdgcn_frexp_mantf(a) * kInverse127 * __builtin_amdgcn_frexp_mantf(s)),
                                   __builtin_amdgcn_frexp_expf(a) + __builtin_amdgcn_frexp_expf(s));
}
// N neighbours of a row
template <int N>
struct Columns8 {
    float step[N], bias[N];
    bool safe;
    __device__ __forceinline__ void init(const float *steps, const Values &b, long n, long D) {
        safe = true;
        if (n + N <= D) {
            // (n is a multiple of four, both vectors are aligned to 16 bytes)
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const mma_f4 q = *reinterpret_cast<const mma_f4 *>(steps + n + e);
#pragma unroll
                for (int k = 0; k < 4; k++) step[e + k] = q[k];
            }
            if (b.p == nullptr) {
#pragma unroll
                for (int e = 0; e < N; e++) bias[e] = 0.f;
            } else if (b.type == OUT_F32) {
#pragma unroll
                for (int e = 0; e < N; e += 4) {
                    const mma_f4 q = *reinterpret_cast<const mma_f4 *>(reinterpret_cast<const float *>(b.p) + n + e);
#pragma unroll
                    for (int k = 0; k < 4; k++) bias[e + k] = q[k];
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; e += 4) {
                    const mma_u2 q = *reinterpret_cast<const mma_u2 *>(reinterpret_cast<const uint16_t *>(b.p) + n + e);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint16_t h = (uint16_t)(q[k / 2] >> (16 * (k % 2)));
                        bias[e + k] = b.type == OUT_F16 ? to_float(__builtin_bit_cast(f16_t, h)) : bf16_value(h);
                    }
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; e++) step[e] = n + e < D ? steps[n + e] : 0.f, bias[e] = b.p != nullptr && n + e < D ? b.at(n + e) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < N; e++) safe = safe && near_one(step[e]);
    }
    // act(..) of four of them, from column `from` on
    __device__ __forceinline__ void finish(int from, mma_i4 sum, float a, int act, mma_f4 &v) const {
#pragma clang fp contract(off)  // (product and sum are rounded each, as where the power of two comes between them)
        if (__builtin_expect(safe && near_one(a), 1)) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = step_value(sum[e], a, step[from + e]) + bias[from + e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = step_value_of_any(sum[e], a, step[from + e]) + bias[from + e];
        }
        if (act >= 0) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = act_value(act, v[e]);
        }
    }
};
// N neighbours (four or eight) of row m, those below D: in pieces of 16, 8 or 4 bytes, as the rows' distance allows
template <int N>
__device__ __forceinline__ void out_row(const Out &o, long m, long n, long D, const mma_f4 (&v)[N / 4]) {
    const bool whole = n + N <= D, aligned = ((uintptr_t)o.p & 15) == 0;
    if (whole && aligned && o.type == OUT_F32 && o.pitch % 4 == 0) {
        mma_f4 *to = reinterpret_cast<mma_f4 *>(reinterpret_cast<float *>(o.p) + (size_t)m * o.pitch + n);
#pragma unroll
        for (int i = 0; i < N / 4; i++) to[i] = v[i];
    } else if (whole && aligned && o.type != OUT_F32 && o.pitch % 2 == 0) {
        uint16_t *to = reinterpret_cast<uint16_t *>(o.p) + (size_t)m * o.pitch + n;
        unsigned w[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; i++) w[i] = pack16(o.type, v[i / 2][2 * (i % 2)], v[i / 2][2 * (i % 2) + 1]);
        if (N == 8 && o.pitch % 8 == 0) {
#pragma unroll
            for (int i = 0; i < N / 8; i++) reinterpret_cast<mma_u4 *>(to)[i] = mma_u4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        } else if (o.pitch % 4 == 0) {
#pragma unroll
            for (int i = 0; i < N / 4; i++) reinterpret_cast<mma_u2 *>(to)[i] = mma_u2{w[2 * i], w[2 * i + 1]};
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; i++) reinterpret_cast<unsigned *>(to)[i] = w[i];
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; e++)
            if (n + e < D) out_one(o, m, n + e, v[e / 4][e % 4]);
    }
}
// The same in tiles, with the power of two by itself for every value: an instruction each, where a second way to go costs the loop in front of it registers
// (and sums that stay in registers, as below, the same code eight times: 16384 x 1024 -> 4096 with GELU 157 us, so 138)
struct Int8Epi {
    static constexpr bool kSums = false, kDirect = false;
    const float *most, *steps;  // of rows of x (a) and of the weight (s)
    Values bias;
    Out out;
    int act;  // -1: none
    struct Lane {
        float step[8], bias[8];
        int e[8];
        bool wide;
    };
    __device__ __forceinline__ Lane begin(const Product &p, long n) const {
        Lane l;
        l.wide = out_wide(out);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float s = n + e < p.N ? steps[n + e] : 0.f;
            l.step[e] = __builtin_amdgcn_frexp_mantf(s), l.e[e] = __builtin_amdgcn_frexp_expf(s);
            l.bias[e] = bias.p != nullptr && n + e < p.N ? bias.at(n + e) : 0.f;
        }
        return l;
    }
    static constexpr int kRow = 1;
    __device__ __forceinline__ unsigned row(const Product &, long m, long, int) const { return __float_as_uint(most[m]); }
    __device__ __forceinline__ Nothing load(const Product &, long, long) const { return {}; }
    __device__ __forceinline__ void octet(const Product &p, const Lane &l, const unsigned *rows, const Nothing &, int, long m, long n,
                                          float (&v)[8]) const {
        if (m >= p.M || n >= p.N) return;
        const float a = __uint_as_float(rows[0]), part = __builtin_amdgcn_frexp_mantf(a) * kInverse127;
        const int ae = __builtin_amdgcn_frexp_expf(a);
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = __builtin_amdgcn_ldexpf((float)__builtin_bit_cast(int, v[e]) * (part * l.step[e]), ae + l.e[e]) + l.bias[e];
        if (act >= 0) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = act_value(act, v[e]);
        }
        out_octet(out, l.wide, m, n, p.N, v);
    }
};

// ------------------------------------------------------------------------------------------------- rows that stay in LDS
struct Resident {
    const int8_t *codes;
    const float *steps;
    Values bias;
    Out out;
    long rows;
    int C, D, act;
    int pitch;          // of the weight's codes
    int depth, stride;  // of a row in LDS: whole rounds of steps, zeros behind the row; and an odd number of sixteen bytes
    int parts, groups;  // of the columns: parts of so many groups
};
// Rows of x from `first` on, `have` of them (ROWS at the most), as codes into LDS, LANES threads a row, up to U pieces a thread; their largest magnitudes
// into `most`.  A thread asks for all its rows, or as many as 64 registers hold, before it waits for one.
template <typename T, int THREADS, int ROWS, int LANES, int U>
__device__ __forceinline__ void rows_to_lds(const T *__restrict__ x, const Resident &q, long first, int have, char *lds, float *most) {
    constexpr int PASS = THREADS / LANES, TURNS = (ROWS + PASS - 1) / PASS, FIT = 32 / (int)sizeof(T) / U, R = TURNS < FIT ? TURNS : FIT < 1 ? 1 : FIT;
    const int l = threadIdx.x % LANES, pieces = q.depth / 8;
    const bool wide = q.C % 8 == 0;
    for (int r0 = (int)threadIdx.x / LANES; r0 < have; r0 += R * PASS) {
        RowPiece<T> v[R][U];
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int u = 0; u < U; u++) {
                v[i][u].clear();
                if (r0 + i * PASS < have && l + u * LANES < pieces) v[i][u].read(x + (first + r0 + i * PASS) * q.C, l + u * LANES, q.C, wide);
            }
        each<R>([&](auto i) {
            const int r = r0 + i * PASS;
            RowMost<T> largest;
#pragma unroll
            for (int u = 0; u < U; u++) largest.meet(v[i][u]);
            const float a = largest.template join<LANES>();
            if (r >= have) return;
            const bool finite = a < INFINITY;
            RowCodes<T> codes;
            codes.init(finite ? a : 0.f);
            if (l == 0) most[r] = finite ? a : NAN;
#pragma unroll
            for (int u = 0; u < U; u++)
                if (l + u * LANES < pieces)
                    reinterpret_cast<mma_u2 *>(lds + r * q.stride)[l + u * LANES] = finite ? piece_codes(codes, v[i][u]) : mma_u2{0u, 0u};
        });
    }
}
// Where a lane reads the weight: index c of fragment i is column n0 + (c / 4) 4 NF + 4 i + c % 4.  What lies behind the last column reads that one,
// what lies behind a row its beginning (the rows in LDS have zeros there).
// Which sixteen bytes of a row are a lane's in step k: two steps share 128 bytes, four lanes have 32 of them each, so that whole lines are read at a time
// (summed indices may come in any order that both operands share)
__device__ __forceinline__ int code_place(int k, int g) { return k / 2 * 128 + g * 32 + k % 2 * 16; }
template <int NF>
struct WeightRows {
    unsigned row[NF];  // (weights of these kernels have fewer bytes)
    __device__ __forceinline__ void seek(const Resident &q, int n0) {
        const int c = threadIdx.x & 15;
#pragma unroll
        for (int i = 0; i < NF; i++) row[i] = (unsigned)min(n0 + c / 4 * 4 * NF + 4 * i + c % 4, q.D - 1) * (unsigned)q.pitch;
    }
    __device__ __forceinline__ void fetch(const Resident &q, int k, mma_s8 (&b)[NF]) const {
        const int at = code_place(k, (threadIdx.x & 63) >> 4);
        const unsigned to = at < q.pitch ? (unsigned)at : 0u;
#pragma unroll
        for (int i = 0; i < NF; i++) b[i] = *reinterpret_cast<const mma_s8 *>(q.codes + (row[i] + to));
    }
};

// Tiles of 64 rows, 32 columns a wave, two steps ahead, two workgroups of eight waves a CU (25088 x 384 -> 1536 with GELU: 54 us, in twice as many of four,
// which make the codes of the same rows twice, 56; 25088 x 96 -> 384 16.3 and 19.9; 64 columns, eight waves a CU: 70; steps further ahead no faster, 32 rows
// 73: each reads the weight once more.  The case's 392 tiles are in one round on 512 places: 136 CUs have two workgroups and 120 have one)
constexpr int kTileRows = 4, kTileColumns = 2, kTileAhead = 2, kTileWaves = 8, kTilePerCu = 2;

// 16 MF rows of x, taken to codes on the way into LDS, times the weight's columns, which come from the caches straight to registers, two steps ahead: a
// wave has 16 NF columns at a time and waits for no other.  The sums' registers hold a row's neighbours: nothing goes through LDS behind them.
template <typename T, int MF, int NF, int LANES, int U, int AHEAD>
__global__ __launch_bounds__(64 * kTileWaves, 4) void int8_resident_kernel(const T *__restrict__ x, Resident q) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float most[16 * MF];
    constexpr int ROWS = 16 * MF;
    // the parts of a tile of rows on one XCD (workgroup ids modulo eight), one behind the other: they read the same rows of x
    const int xcd = (int)blockIdx.x % 8, in = (int)blockIdx.x / 8;
    const long m0 = ((long)(in / q.parts) * 8 + xcd) * ROWS;
    const int part = in % q.parts;
    if (m0 >= q.rows) return;
    const int have = (int)min((long)ROWS, q.rows - m0);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
    const int all = (q.D + 16 * NF - 1) / (16 * NF), end = min((part + 1) * q.groups, all), steps = q.depth / 64;
    int group = part * q.groups + wave;
    WeightRows<NF> w;
    mma_s8 b[AHEAD][NF];
    w.seek(q, group * 16 * NF);
#pragma unroll
    for (int u = 0; u < AHEAD; u++) w.fetch(q, u, b[u]);
    rows_to_lds<T, 64 * kTileWaves, ROWS, LANES, U>(x, q, m0, have, lds, most);
    __syncthreads();
    float a[MF];
    const char *from[MF];  // (rows that are not there read the last one's codes, and are not written)
#pragma unroll
    for (int j = 0; j < MF; j++) {
        const int r = min(16 * j + c, have - 1);
        a[j] = most[r], from[j] = lds + r * q.stride;
    }
    for (; group < end; group += kTileWaves) {
        mma_f4 acc[MF][NF];
#pragma unroll
        for (int j = 0; j < MF; j++)
#pragma unroll
            for (int i = 0; i < NF; i++) acc[j][i] = mma_f4{0.f, 0.f, 0.f, 0.f};
        auto step = [&](int k, int next, mma_s8 (&f)[NF]) {
            mma_s8 rows[MF];
#pragma unroll
            for (int j = 0; j < MF; j++) rows[j] = *reinterpret_cast<const mma_s8 *>(from[j] + code_place(k, g));
#pragma unroll
            for (int j = 0; j < MF; j++)
#pragma unroll
                for (int i = 0; i < NF; i++) acc[j][i] = Mma<i8_t>::run(f[i], rows[j], acc[j][i]);
            w.fetch(q, next, f);
        };
        int k = 0;
        for (; k + AHEAD < steps; k += AHEAD)
#pragma unroll
            for (int u = 0; u < AHEAD; u++) step(k + u, k + u + AHEAD, b[u]);
        w.seek(q, (group + kTileWaves) * 16 * NF);  // (the next group's; behind the last, a column that is there)
#pragma unroll
        for (int u = 0; u < AHEAD; u++) step(k + u, u, b[u]);
        const int n = group * 16 * NF + 4 * NF * g;
        Columns8<4 * NF> l;
        l.init(q.steps, q.bias, n, q.D);
        each<MF>([&](auto j) {  // (one after the other: together they take the registers of all)
            const int r = 16 * j + c;
            if (r >= have || n >= q.D) return;
#pragma unroll
            for (int i = 0; i < NF; i++) {
                const mma_i4 sum = __builtin_bit_cast(mma_i4, acc[j][i]);
                l.finish(4 * i, sum, a[j], q.act, acc[j][i]);
            }
            out_row<4 * NF>(q.out, m0 + r, n, q.D, acc[j]);
        });
    }
}

// Up to sixteen rows times sixteen columns a workgroup: its four waves share the sums, and ask for their part of the weight before the rows' codes are made
template <typename T, int U>
__global__ __launch_bounds__(256, 4) void int8_few_kernel(const T *__restrict__ x, Resident q) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ float most[16];
    __shared__ mma_i4 shares[4 * 64];
    constexpr int AHEAD = 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int n0 = (int)blockIdx.x * 16, have = (int)q.rows, steps = q.depth / 64;
    WeightRows<1> w;
    mma_s8 b[AHEAD][1];
    w.seek(q, n0);
#pragma unroll
    for (int u = 0; u < AHEAD; u++) w.fetch(q, 2 * wave + u / 2 * 8 + u % 2, b[u]);
    rows_to_lds<T, 256, 16, 64, U>(x, q, 0, have, lds, most);
    __syncthreads();
    const int r = min(c, have - 1);
    const char *const from = lds + r * q.stride;
    mma_f4 acc = mma_f4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = 2 * wave; k0 < steps; k0 += 4 * AHEAD)  // (whole rounds; a wave has every fourth pair of steps)
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int k = k0 + u / 2 * 8 + u % 2;
            acc = Mma<i8_t>::run(b[u][0], *reinterpret_cast<const mma_s8 *>(from + code_place(k, g)), acc);
            w.fetch(q, k + 4 * AHEAD, b[u]);
        }
    // whole numbers: in any order
    shares[wave * 64 + lane] = __builtin_bit_cast(mma_i4, acc);
    __syncthreads();
    if (wave != 0) return;
    const mma_i4 sum = (shares[lane] + shares[64 + lane]) + (shares[128 + lane] + shares[192 + lane]);
    const int n = n0 + 4 * g;
    if (c >= have || n >= q.D) return;
    Columns8<4> l;
    l.init(q.steps, q.bias, n, q.D);
    mma_f4 v[1];
    l.finish(0, sum, most[c], q.act, v[0]);
    out_row<4>(q.out, c, n, q.D, v);
}

struct Int8Sizes {
    long rows;
    int C, D, dtype;
    bool ok() const { return rows >= 1 && rows <= 1L << 30 && C >= 1 && C <= 65536 && D >= 1 && D <= 65536 && known(dtype); }
};
// Up to sixteen rows of codes that fit LDS, and a weight whose reading does not take over (bf16, us, as rows of codes and tiles: 1 x 1024 -> 4096 6.8,
// 9.9; 16 x 1024 -> 4096 6.8, 9.9; 1 x 4096 -> 1024 7.7, 12.8; beyond sixteen rows, whose codes every workgroup would make again, 32 x 768 -> 2048 10.7, 9.5; weights of 32 and 64 MB 16 x 1024 -> 32768 16.7,
// 12.4; 1 x 4096 -> 16384 18.6, 17.4)
static bool few_rows(const Int8Sizes &s) {
    return s.rows <= 16 && s.C <= 4096 && s.rows * s.C <= 16384 && s.D * code_pitch(s.C) <= 1L << 24;
}
// Some rows, in tiles of sixteen, whose readings of the weight do not add up to much (bf16 with GELU, us, as rows of codes and larger tiles: 128 x 437 ->
// 2720 7.1, 10.9; 300 x 384 -> 1536 9.2, 9.8; 48 x 2000 -> 500 10.0, 11.2; 800 x 96 -> 384 7.0, 9.6; beyond, 300 x 437 -> 2720 12.3, 11.0; 800 x 384 -> 1536
// 13.3, 10.8; 30000 x 32 -> 64 11.2, in tiles of 64 rows 9.5)
static bool some_rows(const Int8Sizes &s) { return s.rows <= 1 << 14 && s.C <= 2048 && (s.rows + 15) / 16 * s.D * code_pitch(s.C) <= 1L << 24; }
// Many short rows, and a weight not far beyond an XCD's L2 (bf16 with GELU, C -> 4 C, us, as rows of codes and tiles: 1024 x 96 8.4, 10.4; 65536 x 192 51,
// 78; 16384 x 384 33, 47; 4096 x 384 17.8, 17.9 but 1024 x 384 12.1, 11.2; 16384 x 512 46, 62; 4096 x 512 20.8, 19.9; 16384 x 768 -> 2048 60, 68;
// 4096 x 768 -> 2048 25, 23; weights of 4 and 6 MB, with workgroups of four waves, 16384 x 512 -> 8192 217, 262; 16384 x 384 -> 16384 395, 503)
static bool many_short_rows(const Int8Sizes &s) {
    return s.C <= 768 && s.rows >= 10L * s.C && s.rows <= 1L << 24 && s.D * code_pitch(s.C) <= 1L << 23;
}
// Parts of the columns, such that the last of the workgroups ends early: a workgroup's time goes with the columns of its waves, and as much as one group of
// these for its rows (the case above with three workgroups of four waves a CU, in 1, 2, 3, 4 and 6 parts: 71, 77, 59, 67 and 72 us, by this 13, 14, 10, 12
// and 12)
static int resident_parts(long tiles, int groups) {
    int best = 1;
    long least = 0;
    for (int parts = 1; parts <= (groups + kTileWaves - 1) / kTileWaves && (parts == 1 || tiles * parts <= 1L << 21); parts++) {
        const long rounds = (tiles * parts + kLinCus * kTilePerCu - 1) / (kLinCus * kTilePerCu);
        const long t = rounds * (1 + ((groups + parts - 1) / parts + kTileWaves - 1) / kTileWaves);
        if (parts == 1 || t < least) best = parts, least = t;
    }
    return best;
}
template <typename T, int MF, int NF, int LANES, int U, int AHEAD>
static int launch_resident(const Int8Sizes &s, const void *x, Resident q, hipStream_t st) {
    const long tiles = (s.rows + 16 * MF - 1) / (16 * MF);
    const int groups = (s.D + 16 * NF - 1) / (16 * NF), parts = resident_parts(tiles, groups);
    q.groups = ((groups + parts - 1) / parts + kTileWaves - 1) / kTileWaves * kTileWaves, q.parts = (groups + q.groups - 1) / q.groups;
    // (rows an odd number of sixteen bytes apart, so that sixteen rows' pieces lie on different banks)
    q.depth = (q.pitch + 64 * AHEAD - 1) / (64 * AHEAD) * 64 * AHEAD, q.stride = q.depth + 16;
    int8_resident_kernel<T, MF, NF, LANES, U, AHEAD>
        <<<dim3((unsigned)((tiles + 7) / 8 * 8 * q.parts)), dim3(64 * kTileWaves), (size_t)(16 * MF) * q.stride, st>>>((const T *)x, q);
    return status();
}
template <typename T>
static int resident_typed(const Int8Sizes &s, const void *x, Resident q, hipStream_t st) {
    if (few_rows(s)) {
        q.depth = (q.pitch + 1023) / 1024 * 1024, q.stride = q.depth + 16;
        auto *kernel = q.depth <= 1024 ? int8_few_kernel<T, 2> : int8_few_kernel<T, 8>;
        kernel<<<dim3((unsigned)((s.D + 15) / 16)), dim3(256), (size_t)s.rows * q.stride, st>>>((const T *)x, q);
        return status();
    }
    if (some_rows(s)) {
        if (q.pitch <= 512) return launch_resident<T, 1, 1, 32, 2, 4>(s, x, q, st);
        if (q.pitch <= 1024) return launch_resident<T, 1, 1, 32, 4, 4>(s, x, q, st);
        return launch_resident<T, 1, 1, 32, 8, 4>(s, x, q, st);
    }
    if (q.pitch <= 256) return launch_resident<T, kTileRows, kTileColumns, 16, 2, kTileAhead>(s, x, q, st);
    if (q.pitch <= 512) return launch_resident<T, kTileRows, kTileColumns, 16, 4, kTileAhead>(s, x, q, st);
    return launch_resident<T, kTileRows, kTileColumns, 16, 6, kTileAhead>(s, x, q, st);
}

static int int8_linear(const Int8Sizes &s, const void *x, const int8_t *codes, const float *steps, const void *bias, void *y, int act, Arena &ws,
                       hipStream_t st) {
    const long pitch = code_pitch(s.C);
    const bool resident = few_rows(s) || some_rows(s) || many_short_rows(s);
    int8_t *q = (int8_t *)ws.take(resident ? 0 : (size_t)s.rows * pitch);
    float *most = (float *)ws.take(resident ? 0 : (size_t)s.rows * sizeof(float));
    if (ws.dry()) return 0;
    const Out out{y, s.D, 0, s.dtype};
    if (resident) {
        const Resident r{codes, steps, {bias, s.dtype}, out, s.rows, s.C, s.D, act, (int)pitch, 0, 0, 1, 0};
        if (s.dtype == DWO_F32) return resident_typed<float>(s, x, r, st);
        return s.dtype == DWO_BF16 ? resident_typed<bf16_t>(s, x, r, st) : resident_typed<f16_t>(s, x, r, st);
    }
    int e = rows8(x, q, most, s.rows, s.C, s.dtype, true, st);
    if (e) return e;
    const Product p = make_product({q, pitch / 2, 0, 1}, {codes, pitch / 2, 0, 1}, s.rows, s.D, pitch / 2, 0);
    const Int8Epi epi{most, steps, {bias, s.dtype}, out, act};
    return launch_tiles<i8_t, false, false, false>(p, epi, st);
}

}  // namespace dwo

using namespace dwo;

extern "C" {

int dwo_int8_rows(const void *x, void *codes, float *steps, size_t rows, int C, int dtype, void *stream) {
    if (!x || !codes || !steps) return DWO_ERR_NULL_POINTER;
    if (!known(dtype)) return DWO_ERR_BAD_DTYPE;
    if (!Int8Sizes{(long)rows, C, 1, dtype}.ok() || ((uintptr_t)x | (uintptr_t)codes) % 16 != 0 || (uintptr_t)steps % 4 != 0) return DWO_ERR_BAD_SHAPE;
    (void)hipGetLastError();
    return rows8(x, (int8_t *)codes, steps, (long)rows, C, dtype, false, (hipStream_t)stream);
}

size_t dwo_int8_workspace_bytes(size_t rows, int C, int D, int dtype) {
    const Int8Sizes s{(long)rows, C, D, dtype};
    if (!s.ok()) return 0;
    Arena ws = Arena::measure();
    int8_linear(s, nullptr, nullptr, nullptr, nullptr, nullptr, -1, ws, nullptr);
    return ws.used + 256;
}

int dwo_int8_linear(const void *x, const void *codes, const float *steps, const void *bias, void *y, void *ws, size_t ws_bytes, size_t rows,
                    int C, int D, int act, int dtype, void *stream) {
    if (!x || !codes || !steps || !y || !ws) return DWO_ERR_NULL_POINTER;
    if (!known(dtype)) return DWO_ERR_BAD_DTYPE;
    const Int8Sizes s{(long)rows, C, D, dtype};
    if (!s.ok() || act < -1 || act > ACT_SILU || ((uintptr_t)x | (uintptr_t)codes | (uintptr_t)steps | (uintptr_t)bias | (uintptr_t)ws) % 16 != 0)
        return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_int8_workspace_bytes(rows, C, D, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    Arena a{(char *)ws, 0, ws_bytes};
    return int8_linear(s, x, (const int8_t *)codes, steps, bias, y, act, a, (hipStream_t)stream);
}

}  // extern "C"
