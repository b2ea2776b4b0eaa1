// Softmax cross entropy of a linear layer over many classes, without keeping its logits:
//   l = x w^T + b,  lse = log sum_v exp l_v,  loss = lse - (1 - eps) l_t - eps mean_v l_v
//   G = up (exp(l - lse) - (1 - eps) [v = t] - eps / V),  dx = G w,  dw = G^T x,  db = sum over rows of G
//
// Forward: one product over all classes whose epilogue leaves, for a row and a wave's classes, their largest logit and the sum of
// exponentials below it; a second kernel joins them.  Backward, in pieces of the classes: the product again, its sums turned into G, which
// alone goes through memory, rounded to the activations' type (kHalvesWork: to two) for the two products that read it.  Eight operations per
// row, class and channel in place of the six of a pass that keeps its logits; what would be kept is two or more bytes a row and class.
// Bound by the matrix cores: 8192 x 1024 x 65536 in bf16, statistics 1022 us (1075 TFLOP/s), G 4 x 310 (890; 268 MB of G each go out behind
// the sums, which nothing covers), its two products 4 x 460 (1195).  In fp32, 1024 x 512 x 21841: 137, 176 and 323 us, products of six planes at
// 167, 130 and 142 TFLOP/s of the function's own.
#include "dwo_head.h"

namespace dwo {

struct Targets {
    const long long *t;
    long long ignore;
    long V;
    // the class of row m, -1 where the row is ignored, -2 where its target is no class
    __device__ __forceinline__ int of(long m) const {
        const long long v = t[m];
        return v == ignore ? -1 : v >= 0 && v < V ? (int)v : -2;
    }
};

struct StatsEpi {
    static constexpr bool kSums = false, kDirect = true;
    Values bias;
    Targets targets;
    float2 *part;  // [classes / (16 NF)][M]: largest, sum of exponentials
    float *sum;    // the same of sums of logits, or null
    float *at;     // [M]: the target's logit
    static constexpr int kRow = 1;  // the target
    __device__ __forceinline__ unsigned row(const Product &, long m, long, int) const { return (unsigned)targets.of(m); }
    template <int NF>
    __device__ __forceinline__ RowClasses<NF> begin(const Product &p, long n0) const {
        RowClasses<NF> l;
        l.init(bias, n0, p.N);
        return l;
    }
    template <int NF>
    __device__ __forceinline__ void emit(const Product &p, const RowClasses<NF> &l, const unsigned *rows, long m, long n0,
                                         mma_f4 (&v)[NF]) const {
        float most = -INFINITY, s = 0.f;
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) v[i][r] += l.bias[i][r], most = fmaxf(most, v[i][r]);
        if (m < p.M) {
            const int t = (int)rows[0] - (int)class_of(n0, 0, 0);
            if (t >= 0 && t < 16 * NF && (t & 15) < 4) {
                float hit = 0.f;
#pragma unroll
                for (int i = 0; i < NF; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) hit = t == 16 * i + r ? v[i][r] : hit;
                at[m] = hit;
            }
        }
        most = over_lanes(most, [](float a, float b) { return fmaxf(a, b); });
        // (all -infinity: no exponential; NaN is in no maximum and in the sum)
        const float base = most == -INFINITY ? 0.f : most;
        // (exponents are differences here: what rounding their multiples leaves, 2^-24 of each, is small where the term is not)
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) s += __builtin_amdgcn_exp2f((v[i][r] - base) * 1.44269504f);
        s = over_lanes(s, [](float a, float b) { return a + b; });
        const bool writes = (threadIdx.x & 63) < 16 && n0 < p.N && m < p.M;
        const size_t to = (size_t)(n0 / (16 * NF)) * p.M + m;
        if (writes) part[to] = make_float2(most, s);
        if (sum != nullptr) {
            float all = 0.f;
#pragma unroll
            for (int i = 0; i < NF; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) all += class_of(n0, i, r) < p.N ? v[i][r] : 0.f;
            all = over_lanes(all, [](float a, float b) { return a + b; });
            if (writes) sum[to] = all;
        }
    }
};

// place of class t among eight from n on, or one beyond them
__device__ __forceinline__ int place_of(int t, long n) { return t >= (int)n && t < (int)n + 8 ? t - (int)n : 8; }

// The parts of a row joined, K threads a row and R rows at a time; `block` receives a workgroup's sum of losses and number of rows that
// count.  One workgroup with all rows (few of them) writes the mean itself.
// A read of 8 bytes (12 with labels smoothed) a row and part, bound by its latency: four parts a thread are read before the first is joined
// (8192 rows of 1024 parts, 67 MB: 15.3 us, one at a time 32.3).
template <int R, int K>
__global__ __launch_bounds__(R *K) void head_join_kernel(const float2 *__restrict__ part, const float *__restrict__ sum,
                                                           const float *__restrict__ at, Targets targets, float *__restrict__ lse,
                                                           float *__restrict__ loss, float *__restrict__ mean, float *__restrict__ count,
                                                           float2 *__restrict__ block, long M, int parts, float eps) {
    __shared__ float most_of[K][R + 1], sum_of[K][R + 1], all_of[K][R + 1];
    __shared__ float2 rows[R];
    const int r = threadIdx.x % R, k = threadIdx.x / R;
    double total = 0.0, number = 0.0;
    for (long first = (long)blockIdx.x * R; first < M; first += (long)gridDim.x * R) {
        const long m = first + r;
        float most = -INFINITY, s = 0.f, all = 0.f;
        const bool ends = k == 0 && m < M;  // (what the end reads, before the parts)
        const int t = ends ? targets.of(m) : -1;
        const float hit = ends ? at[m] : 0.f;  // (of rows that count)
        if (m < M)
            for (int p = k; p < parts; p += 4 * K) {
                float2 v[4];
                float next = most;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int q = p + K * u;
                    v[u] = q < parts ? part[(size_t)q * M + m] : make_float2(-INFINITY, 0.f);
                    if (sum != nullptr && q < parts) all += sum[(size_t)q * M + m];
                }
#pragma unroll
                for (int u = 0; u < 4; u++) next = fmaxf(next, v[u].x);
                const float base = next == -INFINITY ? 0.f : next;
                s *= below(most - base);
#pragma unroll
                for (int u = 0; u < 4; u++) s += v[u].y * below(v[u].x - base);
                most = next;
            }
        most_of[k][r] = most, sum_of[k][r] = s, all_of[k][r] = all;
        __syncthreads();
        if (k == 0) {
#pragma unroll
            for (int i = 1; i < K; i++) most = fmaxf(most, most_of[i][r]);
            const float base = most == -INFINITY ? 0.f : most;
            s = 0.f, all = 0.f;
#pragma unroll
            for (int i = 0; i < K; i++) s += sum_of[i][r] * below(most_of[i][r] - base), all += all_of[i][r];
            float value = 0.f, counts = 0.f;
            if (m < M) {
                const float l = base + logf(s);
                lse[m] = l;
                if (t == -2) value = NAN;
                else if (t >= 0) value = (l - hit) * (1.f - eps);
                if (t >= 0 && sum != nullptr) value += eps * (l - all / (float)targets.V);
                counts = t != -1 ? 1.f : 0.f;
                if (loss != nullptr) loss[m] = value;
            }
            rows[r] = make_float2(value, counts);
        }
        __syncthreads();
        if (threadIdx.x == 0)
#pragma unroll 16
            for (int i = 0; i < R; i++) total += rows[i].x, number += rows[i].y;
    }
    if (threadIdx.x != 0) return;
    if (block != nullptr) block[blockIdx.x] = make_float2((float)total, (float)number);
    else if (mean != nullptr) mean[0] = (float)(total / number), count[0] = (float)number;
}

// What the products that read G give it back: G is held without what all its rows share.
//   a mean: up / count (1 - eps), so that a row's largest value, about -1 at its target, is next to a number that 16 bits hold; rounded
//   where it is, the same rounding in all rows would go into the gradients (twice their own rounding with labels smoothed)
//   fp16: a power of two besides, or probabilities below 6e-8 would be lost; a mean's values are at most 1 / (1 - eps) and 1 at the target, times
//   2^13 or, above a smoothing of 3/4, what brings 1 / (1 - eps) to 2^14 .. 2^15; others are brought to 2^13 .. 2^14 by the largest finite |up| of a
//   row with a class (whatever arrives at the others changes nothing): scale[0], and its inverse, by head_scale_kernel
static float half_mean_scale(float eps) {
    return eps < 1.f ? fminf(kHalfScale, ldexpf(4.f * kHalfScale, ilogbf(1.f - eps))) : kHalfScale;
}

struct GradEpi {
    static constexpr bool kSums = false, kDirect = false;
    Values bias;      // of the piece
    Targets targets;  // V: all classes
    long from;        // the piece's first class
    const float *lse, *up, *scale;  // up null: a mean; scale null: 1, or a mean's in fp16
    float eps, mean_scale;
    Out g;            // [M][pitch]
    struct Lane : Classes {
        float scale, hit, flat;
    };
    __device__ __forceinline__ Lane begin(const Product &p, long n) const {
        Lane l;
        l.init(bias, n, p.N);
        // (a mean is held without 1 - eps)
        const float s = scale != nullptr ? scale[0] : up == nullptr ? mean_scale : 1.f, part = up == nullptr && eps < 1.f ? s / (1.f - eps) : s;
        l.scale = part, l.hit = up == nullptr && eps < 1.f ? s : s * (1.f - eps), l.flat = part * (eps / (float)targets.V);
        return l;
    }
    static constexpr int kRow = 3;  // the target, the log of the sum, what arrives at the loss
    __device__ __forceinline__ unsigned row(const Product &, long m, long, int k) const {
        return k == 0 ? (unsigned)targets.of(m) : k == 1 ? __float_as_uint(lse[m]) : up != nullptr ? __float_as_uint(up[m]) : 0u;
    }
    __device__ __forceinline__ Nothing load(const Product &, long, long) const { return {}; }
    __device__ __forceinline__ void octet(const Product &p, const Lane &l, const unsigned *rows, const Nothing &, int, long m, long n,
                                          float (&v)[8]) const {
        if (m >= p.M || n >= g.pitch) return;
        const int t = (int)rows[0];
        const float total = __uint_as_float(rows[1]), f = __uint_as_float(rows[2]);
        if (g.plane != 0) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = prod_exp(v[e] + l.bias[e] - total);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = __builtin_amdgcn_exp2f((v[e] + l.bias[e] - total) * 1.44269504f);
        }
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = __builtin_fmaf(v[e], l.scale, -l.flat);
        const int k = place_of(t, from + n);
        if (k < 8) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] -= k == e ? l.hit : 0.f;
        }
        if (up != nullptr) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] *= f;
        }
        // rows that are ignored, or whose target is no class, and columns behind the last class
        if (t < 0 || n + 8 > p.N) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = t == -1 || n + e >= p.N ? 0.f : t == -2 ? NAN : v[e];
        }
        operand_octet(g, m, n, g.pitch, v);
    }
};

static int head_forward(const HeadSizes &s, const void *x, const void *w, const void *b, Targets targets, float eps, float *lse,
                        float *loss, float *count, bool mean, Arena &ws, hipStream_t st) {
    Staging stage;
    const Operand ox = stage.matrix(x, s.rows, s.C, s.dtype, ws), ow = stage.matrix(w, s.V, s.C, s.dtype, ws);
    int e = stage.launch(ws.dry(), st);
    if (e) return e;
    const Product p = make_product(ox, ow, s.rows, s.V, s.C, 0);
    const int width = wave_columns(tile_for(p.M, p.N, p.steps));
    // Up to 128 rows one workgroup joins them all (64 x 1000 classes: 6.3 us, as two launches 4.7 and 2.4); with no more than sixteen parts four
    // threads have a row (32768 x 150 classes: 8.3 us for both launches, sixteen 9.6; 64 rows of 63 parts need the sixteen)
    const int parts = (int)((s.V + width - 1) / width);
    const bool few = s.rows <= 128, narrow = !few && parts <= 16;
    const int group = few || narrow ? 64 : 16;
    const int blocks = few ? 1 : (int)std::min((s.rows + group - 1) / group, 1L << 20);  // (a launch has fewer than 2^32 threads)
    float2 *part = (float2 *)ws.take((size_t)parts * s.rows * sizeof(float2));
    float *sum = eps > 0.f ? (float *)ws.take((size_t)parts * s.rows * sizeof(float)) : nullptr;
    float *at = (float *)ws.take((size_t)s.rows * sizeof(float));
    float2 *block = mean && blocks > 1 ? (float2 *)ws.take((size_t)blocks * sizeof(float2)) : nullptr;
    if (ws.dry()) return 0;
    const StatsEpi epi{{b, s.dtype}, targets, part, sum, at};
    if ((e = launch_product<false, false, false>(p, s.dtype, epi, st))) return e;
    auto *const join = few ? head_join_kernel<64, 16> : narrow ? head_join_kernel<64, 4> : head_join_kernel<16, 16>;
    join<<<dim3((unsigned)blocks), dim3(few ? 1024 : 256), 0, st>>>(part, sum, at, targets, lse, mean ? nullptr : loss, mean ? loss : nullptr,
                                                                    count, block, s.rows, parts, eps);
    if (block != nullptr) head_mean_kernel<<<dim3(1), dim3(1024), 0, st>>>(block, blocks, loss, count);
    return status();
}

static int head_backward(const HeadSizes &s, const float *up, const void *x, const void *w, const void *b, Targets targets, float eps,
                         const float *lse, const float *count, void *dx, void *dw, void *db, int grad, Arena &ws, hipStream_t st) {
    Staging stage;
    const Operand ox = stage.matrix(x, s.rows, s.C, s.dtype, ws), ow = stage.matrix(w, s.V, s.C, s.dtype, ws);
    int e = stage.launch(ws.dry(), st);
    if (e) return e;
    const Operand g = take_operand(ws, s.rows, up8(s.piece()), s.dtype, (double)s.rows * (double)s.C * (double)s.V);
    const bool mean = count != nullptr, half = s.dtype == DWO_F16;
    float *scale = half && !mean ? (float *)ws.take(2 * sizeof(float)) : nullptr;
    if (scale != nullptr && !ws.dry()) {
        head_scale_kernel<<<dim3(1), dim3(1024), 0, st>>>(up, targets, s.rows, scale);
        if ((e = status())) return e;
    }
    const float mean_scale = half ? half_mean_scale(eps) : 1.f;
    auto make = [&](long from, long n, const Operand &wp, const Operand &gp) {
        const GradEpi epi{{b != nullptr ? (const char *)b + from * size_of(s.dtype) : nullptr, s.dtype}, targets, from, lse, mean ? nullptr : up, scale,
                          eps, mean_scale, out_of(gp, s.dtype)};
        return launch_product<false, false, false>(make_product(ox, wp, s.rows, n, s.C, 0), s.dtype, epi, st);
    };
    auto shared = [&](PlainEpi epi) {
        epi.alpha = mean ? up : scale != nullptr ? scale + 1 : nullptr;
        epi.over = count;
        epi.factor = mean ? (eps < 1.f ? 1.f - eps : 1.f) / mean_scale : 1.f;
        return epi;
    };
    return head_pieces(s, ox, ow, g, dx, dw, db, grad, make, shared, ws, st);
}

}  // namespace dwo

using namespace dwo;

extern "C" {

size_t dwo_head_workspace_bytes(size_t rows, int C, int V, int backward, int dtype) {
    const HeadSizes s(rows, C, V, dtype);
    if (!s.ok()) return 0;
    Arena ws = Arena::measure();
    void *const any = (void *)256;  // (nothing is launched)
    const Targets t{(const long long *)any, 0, V};
    if (backward)
        head_backward(s, (const float *)any, any, any, any, t, 0.1f, (const float *)any, nullptr, any, any, any, DWO_F32, ws, nullptr);
    else
        head_forward(s, any, any, any, t, 0.1f, (float *)any, (float *)any, (float *)any, true, ws, nullptr);
    return ws.used + 256;
}

int dwo_head_forward(const void *x, const void *w, const void *bias, const void *targets, long long ignore, float smoothing, float *lse,
                     float *loss, float *count, void *ws, size_t ws_bytes, size_t rows, int C, int V, int dtype, void *stream) {
    if (!x || !w || !targets || !lse || !loss || !ws) return DWO_ERR_NULL_POINTER;
    const HeadSizes s(rows, C, V, dtype);
    if (!known(dtype)) return DWO_ERR_BAD_DTYPE;
    if (!s.ok() || !(smoothing >= 0.f && smoothing <= 1.f) || ((uintptr_t)x | (uintptr_t)w | (uintptr_t)ws) % 16 != 0 ||
        (uintptr_t)targets % 8 != 0)
        return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_head_workspace_bytes(rows, C, V, 0, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    Arena a{(char *)ws, 0, ws_bytes};
    return head_forward(s, x, w, bias, {(const long long *)targets, ignore, s.V}, smoothing, lse, loss, count, count != nullptr, a,
                        (hipStream_t)stream);
}

int dwo_head_backward(const float *up, const void *x, const void *w, const void *bias, const void *targets, long long ignore,
                      float smoothing, const float *lse, const float *count, void *dx, void *dw, void *db, void *ws, size_t ws_bytes,
                      size_t rows, int C, int V, int dtype, int grad_dtype, void *stream) {
    if (!up || !x || !w || !targets || !lse || !ws) return DWO_ERR_NULL_POINTER;
    const HeadSizes s(rows, C, V, dtype);
    if (!known(dtype) || !known(grad_dtype)) return DWO_ERR_BAD_DTYPE;
    if (!s.ok() || !(smoothing >= 0.f && smoothing <= 1.f) || ((uintptr_t)x | (uintptr_t)w | (uintptr_t)ws) % 16 != 0 ||
        (uintptr_t)targets % 8 != 0 || (db && !dw))
        return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_head_workspace_bytes(rows, C, V, 1, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    Arena a{(char *)ws, 0, ws_bytes};
    return head_backward(s, up, x, w, bias, {(const long long *)targets, ignore, s.V}, smoothing, lse, count, dx, dw, db, grad_dtype, a,
                         (hipStream_t)stream);
}

}  // extern "C"
