// What the losses of a linear layer over many classes share (dwo_head.hip, dwo_distill.hip): a lane's classes in an epilogue, the mean over rows,
// the scale of fp16's gradients, and the products that read the logits' gradients piece by piece.
#pragma once

#include <algorithm>
#include <cmath>

#include "dwo_product.h"

namespace dwo {

// bias of the classes n0 + 16 i + 4 g + r that a lane has, -infinity where there is no class: its logit is then no largest one and its
// exponential zero (products with columns that are not there are zeros)
__device__ __forceinline__ long class_of(long n0, int i, int r) { return n0 + 16 * i + 4 * ((threadIdx.x & 63) >> 4) + r; }
template <int NF>
struct RowClasses {
    float bias[NF][4];
    __device__ __forceinline__ void init(const Values &b, long n0, long N) {
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const long n = class_of(n0, i, r);
                bias[i][r] = n >= N ? -INFINITY : b.p != nullptr ? b.at(n) : 0.f;
            }
    }
};
// joined over the four lanes that have a row
template <class F>
__device__ __forceinline__ float over_lanes(float v, F &&join) {
    const unsigned u = __float_as_uint(v);
    const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned w = __float_as_uint(join(__uint_as_float(s[0]), __uint_as_float(s[1])));
    const auto t = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return join(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

// bias of the eight classes that a lane has, -infinity where there is no class: its logit is then no largest one and its exponential zero
// (products with columns that are not there are zeros)
struct Classes {
    float bias[8];
    __device__ __forceinline__ void init(const Values &b, long n, long N) {
#pragma unroll
        for (int e = 0; e < 8; e++) bias[e] = n + e >= N ? -INFINITY : b.p != nullptr ? b.at(n + e) : 0.f;
    }
};

// exp of what a logit is below another: the multiple's rounding is 2^-24 of the difference, which is at most the log of a part's width where
// the part counts
__device__ __forceinline__ float below(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504f); }

// The same of many workgroups' sums, in a fixed order and in 64 bits
static __global__ __launch_bounds__(1024) void head_mean_kernel(const float2 *__restrict__ block, int blocks, float *__restrict__ loss,
                                                         float *__restrict__ count) {
    __shared__ double value[1024], number[1024];
    double a = 0.0, b = 0.0;
    for (int i = threadIdx.x; i < blocks; i += 1024) a += block[i].x, b += block[i].y;
    value[threadIdx.x] = a, number[threadIdx.x] = b;
    __syncthreads();
    for (int half = 512; half > 0; half >>= 1) {
        if ((int)threadIdx.x < half)
            value[threadIdx.x] += value[threadIdx.x + half], number[threadIdx.x] += number[threadIdx.x + half];
        __syncthreads();
    }
    if (threadIdx.x == 0) loss[0] = (float)(value[0] / number[0]), count[0] = (float)number[0];
}

// fp16's power of two for rows of which each has a gradient of its own to arrive, by the largest finite |up| of a row that counts
// (rows.of(m) >= 0; whatever arrives at the others changes nothing): scale[0] brings it to 2^13 .. 2^14, scale[1] is its inverse
constexpr float kHalfScale = 8192.f;
template <class Rows>
__global__ __launch_bounds__(1024) void head_scale_kernel(const float *__restrict__ up, Rows targets, long M,
                                                          float *__restrict__ scale) {
    __shared__ unsigned most[1024];
    unsigned v = 0;
    // (one workgroup, bound by the reads' latency: eight rows of a thread are asked for at once; 10^6 rows 170 us, one at a time 610)
    for (long i = threadIdx.x; i < M; i += 8 * 1024) {
        unsigned u[8];
        int t[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const long m = min(i + 1024 * k, M - 1);
            u[k] = __float_as_uint(up[m]) & 0x7fffffffu, t[k] = targets.of(m);
        }
#pragma unroll
        for (int k = 0; k < 8; k++) v = u[k] < 0x7f800000u && t[k] >= 0 ? max(v, u[k]) : v;
    }
    most[threadIdx.x] = v;
    __syncthreads();
    for (int h = 512; h > 0; h >>= 1) {
        if ((int)threadIdx.x < h) most[threadIdx.x] = max(most[threadIdx.x], most[threadIdx.x + h]);
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const int e = (int)(most[0] >> 23);  // biased exponent; the scale's is 254 + 13 - e
        const int k = e == 0 ? 127 : min(max(267 - e, 1), 253);
        scale[0] = __uint_as_float((unsigned)k << 23), scale[1] = __uint_as_float((unsigned)(254 - k) << 23);
    }
}

struct HeadSizes {
    long rows, C, V;
    int dtype;
    HeadSizes(size_t r, int c, int v, int t) : rows((long)r), C(c), V(v), dtype(t) {}
    bool ok() const { return rows >= 1 && rows <= 1L << 30 && C >= 1 && C <= 65536 && V >= 1 && V <= 1 << 24 && known(dtype); }
    // classes of a piece: G of a piece has about 2^27 values, 256 MB in 16 bits, what the last cache before memory holds, or 1024 classes
    long piece() const {
        const long most = std::max((1L << 27) / rows / 256 * 256, 1024L);
        return std::min(V, most);
    }
};

// dx, dw and db from the logits' gradients G, made in pieces of the classes: make(from, n, w, g) leaves those of n classes in operand g, and
// shared(epilogue) is what the products that read it give it back.  Both in one launch, or apart: each is then split and in tiles as suits it alone.
template <class Make, class Shared>
int head_pieces(const HeadSizes &s, const Operand &ox, const Operand &ow, const Operand &g, void *dx, void *dw, void *db, int grad, Make &&make,
                Shared &&shared, Arena &ws, hipStream_t st, bool apart = false) {
    const long piece = s.piece();
    // dx is summed over the pieces in fp32
    const bool many = piece < s.V;
    float *sum = many && dx != nullptr && s.dtype != DWO_F32 ? (float *)ws.take((size_t)s.rows * s.C * sizeof(float)) : (float *)dx;
    const size_t grad_size = size_of(grad), held = ws.used;
    size_t peak = held;
    int e = 0;
    for (long from = 0; from < s.V; from += piece) {
        const long n = s.V - from < piece ? s.V - from : piece;
        ws.used = held;  // (the pieces' partial sums take the same place)
        Operand wp = ow;
        wp.p = (const char *)ow.p + (size_t)from * ow.pitch * 2;
        Operand gp = g;
        gp.pitch = up8(n), gp.plane = s.rows * gp.pitch;
        if (!ws.dry() && (e = make(from, n, wp, gp))) return e;
        ProductGroup group;
        if (dx != nullptr) {
            const bool last = from + n == s.V;
            PlainEpi epi = shared(plain_epilogue({last ? dx : (void *)sum, s.C, 0, last ? s.dtype : (int)OUT_F32}));
            epi.before = from > 0 ? sum : nullptr;
            group.add(false, gp, wp, s.rows, s.C, n, epi);
            if (apart) {
                if ((e = group.launch(s.dtype, ws, st))) return e;
                if (ws.used > peak) peak = ws.used;
                ws.used = held, group = ProductGroup{};
            }
        }
        if (dw != nullptr) {
            PlainEpi epi = shared(plain_epilogue({(char *)dw + (size_t)from * s.C * grad_size, s.C, 0, grad}));
            epi.sums = {db != nullptr ? (char *)db + from * grad_size : nullptr, 0, 0, grad};
            group.add(true, gp, ox, n, s.C, s.rows, epi);
        }
        if ((e = group.launch(s.dtype, ws, st))) return e;
        if (ws.used > peak) peak = ws.used;
    }
    ws.used = peak;
    return 0;
}

}  // namespace dwo
