// Linear layers at inference as products of 8-bit integers:
//   q = round(127 x / a), a the row's largest magnitude;  y = act((sum_c q_c p_c) (a / 127) s + b) for weights held as codes p and steps s.
//
// A pass over x that leaves its codes and every row's a, and a product whose epilogue does the rest.  Whole numbers are summed, below 2^30 for 65536
// channels: sums are exact and in any order.
#include "dwo_act.h"
#include "dwo_int8.h"

namespace dwo {

constexpr int kCodePiece = 16;  // rows of codes are filled up to whole sixteen bytes
static long code_pitch(long C) { return (C + kCodePiece - 1) / kCodePiece * kCodePiece; }

// Codes of rows, LANES of a workgroup's threads a row, U pieces of eight values a lane (0: any number, read twice).  steps: a / 127 of each row or, for
// the product that follows, a itself; NaN where a value of the row is not finite, its codes are then zero.
template <typename T, int LANES, int U>
__global__ __launch_bounds__(256) void rows8_kernel(const T *__restrict__ x, int8_t *__restrict__ codes, float *__restrict__ steps, long rows,
                                                    int C, long pitch, bool raw) {
    __shared__ unsigned part[4];
    constexpr int ROWS = 256 / LANES;
    const int lane = threadIdx.x % LANES, pieces = (int)(pitch / 8);
    const bool wide = C % 8 == 0;
    for (long first = (long)blockIdx.x * ROWS; first < rows; first += (long)gridDim.x * ROWS) {
        const long row = first + threadIdx.x / LANES;
        const T *at = x + row * C;
        auto read = [&](int piece, float (&v)[8]) {
            const int c = piece * 8;
            if (row < rows && wide && c < C) {
                mma_u4 w[sizeof(T) / 2];
#pragma unroll
                for (int k = 0; k < (int)sizeof(T) / 2; k++) w[k] = reinterpret_cast<const mma_u4 *>(at + c)[k];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = to_float(reinterpret_cast<const T *>(w)[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = row < rows && c + e < C ? to_float(at[c + e]) : 0.f;
            }
        };
        unsigned most = 0;
        auto meet = [&](const float (&v)[8]) {
#pragma unroll
            for (int e = 0; e < 8; e++) most = max(most, __float_as_uint(v[e]) & 0x7fffffffu);
        };
        float v[U > 0 ? U : 1][8];
        if constexpr (U > 0) {
#pragma unroll
            for (int u = 0; u < U; u++) read(lane + u * LANES, v[u]);
#pragma unroll
            for (int u = 0; u < U; u++) meet(v[u]);
        } else {
            for (int p = lane; p < pieces; p += LANES) read(p, v[0]), meet(v[0]);
        }
#pragma unroll
        for (int off = 1; off < (LANES < 64 ? LANES : 64); off <<= 1) most = max(most, (unsigned)__shfl_xor((int)most, off, 64));
        if constexpr (LANES > 64) {
            __syncthreads();
            if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = most;
            __syncthreads();
            most = max(max(part[0], part[1]), max(part[2], part[3]));
        }
        if (row >= rows) continue;  // (with LANES above 64 no row is)
        const bool finite = finite_bits(most);
        const float a = __uint_as_float(most);
        RowCodes<T> r;
        r.init(finite ? a : 0.f);
        if (lane == 0) steps[row] = !finite ? NAN : raw ? a : a / 127.f;
        auto write = [&](int piece, const float (&value)[8]) {
            mma_u2 w = mma_u2{0u, 0u};
            if (finite)
#pragma unroll
                for (int e = 0; e < 8; e++) w[e / 4] |= (unsigned)(r.code(value[e]) & 0xff) << (8 * (e % 4));
            reinterpret_cast<mma_u2 *>(codes + row * pitch)[piece] = w;
        };
        if constexpr (U > 0) {
#pragma unroll
            for (int u = 0; u < U; u++)
                if (lane + u * LANES < pieces) write(lane + u * LANES, v[u]);
        } else {
            for (int p = lane; p < pieces; p += LANES) read(p, v[0]), write(p, v[0]);
        }
    }
}

template <typename T>
static int launch_rows8(const void *x, int8_t *codes, float *steps, long rows, int C, bool raw, hipStream_t st) {
    const long pitch = code_pitch(C);
    auto go = [&](auto *kernel, int lanes) {
        const long per = 256 / lanes, blocks = (rows + per - 1) / per;
        kernel<<<dim3((unsigned)(blocks < 1L << 20 ? blocks : 1L << 20)), dim3(256), 0, st>>>((const T *)x, codes, steps, rows, C, pitch, raw);
    };
    if (pitch <= 128) go(rows8_kernel<T, 16, 1>, 16);
    else if (pitch <= 512) go(rows8_kernel<T, 64, 1>, 64);
    else if (pitch <= 2048) go(rows8_kernel<T, 64, 4>, 64);
    else if (pitch <= 8192) go(rows8_kernel<T, 256, 4>, 256);
    else go(rows8_kernel<T, 256, 0>, 256);
    return status();
}
static int rows8(const void *x, int8_t *codes, float *steps, long rows, int C, int dtype, bool raw, hipStream_t st) {
    if (dtype == DWO_F32) return launch_rows8<float>(x, codes, steps, rows, C, raw, st);
    if (dtype == DWO_BF16) return launch_rows8<bf16_t>(x, codes, steps, rows, C, raw, st);
    return launch_rows8<f16_t>(x, codes, steps, rows, C, raw, st);
}

constexpr float kInverse127 = 1.f / 127.f;
// a s / 127 as a number near 1 and a power of two, so that neither factor's size costs digits or is infinite where the result is not
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
            l.step[e] = __builtin_amdgcn_frexp_mantf(s) * kInverse127, l.e[e] = __builtin_amdgcn_frexp_expf(s);
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
        const float a = __uint_as_float(rows[0]), am = __builtin_amdgcn_frexp_mantf(a);
        const int ae = __builtin_amdgcn_frexp_expf(a);
#pragma unroll
        for (int e = 0; e < 8; e++)
            v[e] = __builtin_amdgcn_ldexpf((float)__builtin_bit_cast(int, v[e]) * (am * l.step[e]), ae + l.e[e]) + l.bias[e];
        if (act >= 0) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = act_value(act, v[e]);
        }
        out_octet(out, l.wide, m, n, p.N, v);
    }
};

struct Int8Sizes {
    long rows;
    int C, D, dtype;
    bool ok() const { return rows >= 1 && rows <= 1L << 30 && C >= 1 && C <= 65536 && D >= 1 && D <= 65536 && known(dtype); }
};
static int int8_linear(const Int8Sizes &s, const void *x, const int8_t *codes, const float *steps, const void *bias, void *y, int act, Arena &ws,
                       hipStream_t st) {
    const long pitch = code_pitch(s.C);
    int8_t *q = (int8_t *)ws.take((size_t)s.rows * pitch);
    float *most = (float *)ws.take((size_t)s.rows * sizeof(float));
    if (ws.dry()) return 0;
    int e = rows8(x, q, most, s.rows, s.C, s.dtype, true, st);
    if (e) return e;
    const Product p = make_product({q, pitch / 2, 0, 1}, {codes, pitch / 2, 0, 1}, s.rows, s.D, pitch / 2, 0);
    const Int8Epi epi{most, steps, {bias, s.dtype}, {y, s.D, 0, s.dtype}, act};
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
    if (!s.ok() || act < -1 || act > ACT_SILU || ((uintptr_t)x | (uintptr_t)codes | (uintptr_t)ws) % 16 != 0 || (uintptr_t)steps % 4 != 0)
        return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_int8_workspace_bytes(rows, C, D, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    Arena a{(char *)ws, 0, ws_bytes};
    return int8_linear(s, x, (const int8_t *)codes, steps, bias, y, act, a, (hipStream_t)stream);
}

}  // extern "C"
