// The loss of a linear layer over many classes against a teacher's top logits, without keeping its own logits.  Row m has entries j: a class c_j and the
// teacher's logit t_j; those of class -1, or whose logit is -infinity, are absent.
//   p = softmax over the entries that are there of t / T,  l = x w^T + b,  q = softmax over all classes of l / T
//   loss = T^2 sum_j p_j (log p_j - log q_{c_j}),  G_v = up T (q_v - sum over j with c_j = v of p_j),  dx = G w,  dw = G^T x,  db = sum over rows of G
// A row without entries has no loss, no gradient, and does not count in the mean.
//
// A first pass makes each row's distribution, with its entries in the order of their classes, and a table that says for each run of 64 classes which
// entries lie in it: so the product over all classes, whose epilogue leaves the statistics of l (dwo_head.hip), finds the few sums that are some
// entry's logit among its own and leaves them too.  (Where most runs have several entries it leaves all its sums instead.)  Backward, in
// pieces of the classes: the product again, its sums turned into up T q; a pass over the entries then puts up T (q - p) in their places, computed from
// the logits left by the forward pass in fp32 and rounded once.
//
// Of a row's statistics both numbers are kept, the largest logit m and s = sum exp((l - m) / T): q = exp((l - m) / T) / s.  One number, m + T log s,
// would be rounded at the size of the logits, and 1 / T times that is an error of all of a row's q (logits of 64, T = 0.001: 0.4 %).
#include "dwo_head.h"

namespace dwo {

typedef int mma_i4 __attribute__((ext_vector_type(4)));

constexpr int kDistillMost = 1024;  // entries of a row
constexpr int kNowhere = 1 << 30;   // an absent entry's class is this and its place: no two are the same
constexpr int kRun = 64;            // classes of a word of the table, no fewer than a wave's columns in any tile
// A run's word: the first entry's place in the run, its place among the row's entries, and how many there are
__device__ __forceinline__ unsigned run_word(int place, int start, int count) { return (unsigned)place | (unsigned)start << 6 | (unsigned)count << 16; }
__device__ __forceinline__ int run_place(unsigned w) { return w & 63; }
__device__ __forceinline__ int run_start(unsigned w) { return w >> 6 & 1023; }
__device__ __forceinline__ int run_count(unsigned w) { return w >> 16; }
static long run_pitch(long V) { return ((V + kRun - 1) / kRun + 3) / 4 * 4; }

// A row's state: without entries; a class that is none or a logit that is no number; of others 0, and from the join on the bits of its largest logit
// (0 where all are -infinity), which is never NaN, as these two are
enum { ROW_OUT = -1, ROW_BAD = -2 };
__device__ __forceinline__ bool row_odd(int state) { return state == ROW_OUT || state == ROW_BAD; }
struct RowStates {
    const int *state;
    __device__ __forceinline__ int of(long m) const { return row_odd(state[m]) ? -1 : 0; }
};
// what the backward pass takes of the forward one: [M][k] each but the last two, [M]
struct Kept {
    int *classes;  // in order, absent ones behind the others
    float *p, *at;  // and the layer's logit there (not written for absent ones)
    int *state;
    float *sum;  // of exp((l - the largest) / T)
    Kept(float *keep, long rows, int k) {
        const size_t all = (size_t)rows * k;
        classes = (int *)keep, p = keep + all, at = keep + 2 * all, state = (int *)(keep + 3 * all), sum = keep + 3 * all + rows;
    }
};

// ------------------------------------------------------------------------------------------------- the teacher's entries
// G lanes a row, N entries a lane (j = lane + G i).  An entry's place in the order of classes is the number of those in front of it; entries of one
// class, which are rare, stay in their order.  (8192 rows of 64 entries, 65536 classes: 14 us, 33 MB of them the table; each row's words are written as
// zeros, and those of its runs again.  Of many entries their comparisons bound it, two instructions for each pair.)
template <typename T, int G, int N>
__global__ __launch_bounds__(256) void distill_entries_kernel(const T *__restrict__ logits, const long long *__restrict__ classes, Kept kept,
                                                              unsigned *__restrict__ table, long rows, long V, int k, long pitch, float per) {
    constexpr int ROWS = 256 / G;
    constexpr int PITCH = G * N + 4;  // (rows of a wave on different banks)
    __shared__ __attribute__((aligned(16))) int lds[ROWS][PITCH];
    const int lane = threadIdx.x % G;
    int *const mine = lds[threadIdx.x / G];
    auto join = [](float v, auto &&f) {
#pragma unroll
        for (int off = 1; off < G; off <<= 1) v = f(v, __shfl_xor(v, off, 64));
        return v;
    };
    for (long first = (long)blockIdx.x * ROWS; first < rows; first += (long)gridDim.x * ROWS) {
        const long row = first + threadIdx.x / G;
        const bool real = row < rows;
        float t[N];
        int c[N];
        float bad = 0.f, most = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int j = lane + G * i;
            t[i] = -INFINITY, c[i] = kNowhere + j;
            if (real && j < k) {
                const long long v = classes[row * k + j];
                const float f = to_float(logits[row * k + j]);
                const bool is = v >= 0 && v < V;
                if (v != -1 && f != -INFINITY && (!is || !(f < INFINITY))) bad = 1.f;
                if (is && f != -INFINITY) t[i] = f, c[i] = (int)v;
            }
            most = fmaxf(most, t[i]);
            mine[j] = c[i];
        }
        if (real && table != nullptr)
            for (long b = lane; b < pitch / 4; b += G) reinterpret_cast<mma_u4 *>(table + row * pitch)[b] = mma_u4{0u, 0u, 0u, 0u};
        const bool any_bad = join(bad, [](float a, float b) { return fmaxf(a, b); }) != 0.f;
        most = join(most, [](float a, float b) { return fmaxf(a, b); });
        const bool some = most > -INFINITY;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            t[i] = some && !any_bad && t[i] > -INFINITY ? prod_exp((t[i] - most) * per) : 0.f;
            sum += t[i];
        }
        sum = join(sum, [](float a, float b) { return a + b; });
        const float part = some && !any_bad ? 1.f / sum : 0.f;
        if (real && lane == 0) kept.state[row] = any_bad ? ROW_BAD : some ? 0 : ROW_OUT;
        __syncthreads();  // (the classes are in LDS)
        int rank[N] = {}, ranks = 0;
        for (int j = 0; j < k; j += 4) {  // (what is behind the last entry is above all)
            const mma_i4 other = *reinterpret_cast<const mma_i4 *>(mine + j);
#pragma unroll
            for (int h = 0; h < 4; h++)
#pragma unroll
                for (int i = 0; i < N; i++) rank[i] += other[h] < c[i] ? 1 : 0;
        }
#pragma unroll
        for (int i = 0; i < N; i++) ranks += lane + G * i < k ? rank[i] : 0;
#pragma unroll
        for (int off = 1; off < G; off <<= 1) ranks += __shfl_xor(ranks, off, 64);
        // (0 .. k - 1 unless two are the same)
        if (__any(ranks != k * (k - 1) / 2))
            for (int j = 0; j < k; j++) {
                const int other = mine[j];
#pragma unroll
                for (int i = 0; i < N; i++) rank[i] += other == c[i] && j < lane + G * i ? 1 : 0;
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; i++)
            if (lane + G * i < k) mine[rank[i]] = c[i];
        __syncthreads();  // (in order; and the zeros are in memory in front of the words that replace some)
#pragma unroll
        for (int i = 0; i < N; i++)
            if (real && lane + G * i < k) {
                const int at = rank[i], run = c[i] / kRun;
                kept.classes[row * k + at] = c[i];
                kept.p[row * k + at] = t[i] * part;
                if (table != nullptr && c[i] < kNowhere && (at == 0 || mine[at - 1] / kRun != run)) {
                    int count = 1;
                    while (at + count < k && mine[at + count] / kRun == run) count++;
                    table[row * pitch + run] = run_word(c[i] % kRun, at, count);
                }
            }
        __syncthreads();
    }
}
template <typename T>
static int launch_entries(const void *logits, const long long *classes, const Kept &kept, unsigned *table, long rows, long V, int k, float per,
                          hipStream_t st) {
    auto go = [&](auto *kernel, int lanes) {
        const long each = 256 / lanes, blocks = (rows + each - 1) / each;
        kernel<<<dim3((unsigned)std::min(blocks, 1L << 20)), dim3(256), 0, st>>>((const T *)logits, classes, kept, table, rows, V, k, run_pitch(V), per);
    };
    if (k <= 8) go(distill_entries_kernel<T, 8, 1>, 8);
    else if (k <= 16) go(distill_entries_kernel<T, 16, 1>, 16);
    else if (k <= 32) go(distill_entries_kernel<T, 32, 1>, 32);
    else if (k <= 64) go(distill_entries_kernel<T, 64, 1>, 64);
    else if (k <= 128) go(distill_entries_kernel<T, 64, 2>, 64);
    else if (k <= 256) go(distill_entries_kernel<T, 64, 4>, 64);
    else go(distill_entries_kernel<T, 64, 16>, 64);
    return status();
}

// ------------------------------------------------------------------------------------------------- statistics
struct DistillStatsEpi {
    static constexpr bool kSums = false, kDirect = true;
    Values bias;
    const unsigned *table;
    long pitch;
    const int *classes;
    int k;
    float *at;     // [M][k]
    float *all;    // or all logits, [M][up4(V)], and no table
    float2 *part;  // [classes / (16 NF)][M]: largest logit, sum of exponentials of those / T below it
    float scale;   // log2(e) / T
    static constexpr int kRow = 4;  // the words of the 256 classes around the tile
    __device__ __forceinline__ unsigned row(const Product &, long m, long n0, int i) const {
        const long b = n0 / (4 * kRun) * 4 + i;
        return table != nullptr && b < pitch ? table[m * pitch + b] : 0u;
    }
    template <int NF>
    __device__ __forceinline__ RowClasses<NF> begin(const Product &p, long n0) const {
        RowClasses<NF> l;
        l.init(bias, n0, p.N);
        return l;
    }
    // v[t / 16][t % 4], by the bits of t
    template <int NF>
    static __device__ __forceinline__ float pick(const mma_f4 (&v)[NF], int t) {
        float w[NF];
#pragma unroll
        for (int i = 0; i < NF; i++) {
            const float lo = t & 1 ? v[i][1] : v[i][0], hi = t & 1 ? v[i][3] : v[i][2];
            w[i] = t & 2 ? hi : lo;
        }
#pragma unroll
        for (int n = NF / 2, bit = 16 * n; n > 0; n /= 2, bit /= 2)
#pragma unroll
            for (int i = 0; i < n; i++) w[i] = t & bit ? w[i + n] : w[i];
        return w[0];
    }
    template <int NF>
    __device__ __forceinline__ void emit(const Product &p, const RowClasses<NF> &l, const unsigned *rows, long m, long n0,
                                         mma_f4 (&v)[NF]) const {
        static_assert(16 * NF <= kRun, "a wave's columns are in one run");
        float most = -INFINITY, s = 0.f;
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) v[i][r] += l.bias[i][r], most = fmaxf(most, v[i][r]);
        if (all != nullptr && m < p.M)
#pragma unroll
            for (int i = 0; i < NF; i++) {
                const long n = class_of(n0, i, 0), wide = (p.N + 3) / 4 * 4;
                if (n < wide) *reinterpret_cast<mma_f4 *>(all + m * wide + n) = v[i];
            }
        const unsigned word = rows[n0 / kRun % 4];
        if (m < p.M && word != 0) {
            const int lane_class = (int)class_of(n0, 0, 0), start = run_start(word), count = run_count(word);
            auto hit = [&](int t, int j) {
                if (t >= 0 && t < 16 * NF && (t & 15) < 4) at[m * k + start + j] = pick(v, t);
            };
            hit((int)(n0 / kRun) * kRun + run_place(word) - lane_class, 0);
            for (int j = 1; j < count; j += 4) {  // (of few classes many a run has several: four are asked for at a time)
                int c[4];
#pragma unroll
                for (int u = 0; u < 4; u++) c[u] = classes[m * k + start + min(j + u, count - 1)];
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (j + u < count) hit(c[u] - lane_class, j + u);
            }
        }
        most = over_lanes(most, [](float a, float b) { return fmaxf(a, b); });
        // (all -infinity: no exponential; NaN is in no maximum and in the sum)
        const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
        for (int i = 0; i < NF; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) s += __builtin_amdgcn_exp2f((v[i][r] - base) * scale);
        s = over_lanes(s, [](float a, float b) { return a + b; });
        if ((threadIdx.x & 63) < 16 && n0 < p.N && m < p.M) part[(size_t)(n0 / (16 * NF)) * p.M + m] = make_float2(most, s);
    }
};

// The parts of a row joined and its loss, K threads a row and R rows at a time; a workgroup's sum and number go to `block`, or with all rows in one it
// writes the mean itself (as head_join_kernel).  With sixteen rows the four threads that a wave has of each are joined first.  (1024 rows of 342
// parts: 64 threads a row 7.9 us, 16 of them 11.6; 8192 rows of 1024 parts, 67 MB, 17 either way: memory.)
template <int R, int K>
__global__ __launch_bounds__(R *K) void distill_join_kernel(const float2 *__restrict__ part, Kept kept, float *__restrict__ loss,
                                                            float *__restrict__ mean, float *__restrict__ count, float2 *__restrict__ block,
                                                            const float *__restrict__ all, long wide, long M, int parts, int entries, float T) {
    constexpr int FOUR = R == 16 ? 4 : 1, W = K / FOUR;
    __shared__ float most_of[W][R + 1], sum_of[W][R + 1];
    __shared__ float2 rows[R];
    const int r = threadIdx.x % R, k = threadIdx.x / R, w = k / FOUR;
    const float per = 1.f / T, scale = 1.44269504f * per;
    auto larger = [](float a, float b) { return fmaxf(a, b); };
    auto total_of = [](float a, float b) { return a + b; };
    double total = 0.0, number = 0.0;
    for (long first = (long)blockIdx.x * R; first < M; first += (long)gridDim.x * R) {
        const long m = first + r;
        float most = -INFINITY, s = 0.f;
        const int state = m < M ? kept.state[m] : (int)ROW_OUT;
        // (to a base that is a number: all -infinity has no exponential)
        auto rebase = [&](float next) {
            const float base = next == -INFINITY ? 0.f : next;
            s *= __builtin_amdgcn_exp2f((most - base) * scale);
            most = next;
            return base;
        };
        if (m < M)
            for (int p = k; p < parts; p += 4 * K) {
                float2 v[4];
                float next = most;
#pragma unroll
                for (int u = 0; u < 4; u++) v[u] = p + K * u < parts ? part[(size_t)(p + K * u) * M + m] : make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int u = 0; u < 4; u++) next = fmaxf(next, v[u].x);
                const float base = rebase(next);
#pragma unroll
                for (int u = 0; u < 4; u++) s += v[u].y * __builtin_amdgcn_exp2f((v[u].x - base) * scale);
            }
        if constexpr (FOUR > 1) {
            rebase(over_lanes(most, larger));
            s = over_lanes(s, total_of);
        }
        most_of[w][r] = most, sum_of[w][r] = s;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; i++) most = fmaxf(most, most_of[i][r]);
        const float base = most == -INFINITY ? 0.f : most;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < W; i++) s += sum_of[i][r] * __builtin_amdgcn_exp2f((most_of[i][r] - base) * scale);
        const float log_sum = logf(s);
        __syncthreads();
        // sum of p (log p - log q): both logarithms are of one size where the layer follows the teacher
        float value = 0.f;
        if (state == 0)
            for (int j = k; j < entries; j += K) {
                const float p = kept.p[m * entries + j];
                float l = 0.f;
                if (all != nullptr) {
                    const int c = kept.classes[m * entries + j];
                    if (c < kNowhere) kept.at[m * entries + j] = l = all[m * wide + c];
                } else if (p > 0.f) {
                    l = kept.at[m * entries + j];
                }
                if (p > 0.f) value = __builtin_fmaf(p, logf(p) - ((l - base) * per - log_sum), value);
            }
        if constexpr (FOUR > 1) value = over_lanes(value, total_of);
        sum_of[w][r] = value;
        __syncthreads();
        if (k == 0) {
#pragma unroll
            for (int i = 1; i < W; i++) value += sum_of[i][r];
            value = state == ROW_OUT ? 0.f : state == ROW_BAD ? NAN : T * T * value;
            if (m < M) {
                kept.sum[m] = s;
                if (state == 0) kept.state[m] = __float_as_int(base);
                if (loss != nullptr) loss[m] = value;
            }
            rows[r] = make_float2(value, state != ROW_OUT ? 1.f : 0.f);
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

// ------------------------------------------------------------------------------------------------- gradients of the logits
// q times what each row's loss receives, without what all rows share (T, and a mean's up / count); in fp16 times a power of two, as dwo_head.hip has it
struct DistillGrad {
    const int *state;
    const float *sum, *up, *scale;  // up null: a mean; scale null: `fixed`
    float per, fixed;               // 1 / T
    __device__ __forceinline__ float factor(long m) const { return (up != nullptr ? up[m] : 1.f) * (scale != nullptr ? scale[0] : fixed); }
};
struct DistillGradEpi {
    static constexpr bool kSums = false, kDirect = false;
    Values bias;  // of the piece
    DistillGrad d;
    Out g;  // [M][pitch]
    using Lane = Classes;
    __device__ __forceinline__ Lane begin(const Product &p, long n) const {
        Lane l;
        l.init(bias, n, p.N);
        return l;
    }
    static constexpr int kRow = 2;  // the state, or largest logit; what arrives at the loss, over the sum
    __device__ __forceinline__ unsigned row(const Product &, long m, long, int k) const {
        return k == 0 ? (unsigned)d.state[m] : __float_as_uint(d.factor(m) / d.sum[m]);
    }
    __device__ __forceinline__ Nothing load(const Product &, long, long) const { return {}; }
    __device__ __forceinline__ void octet(const Product &p, const Lane &l, const unsigned *rows, const Nothing &, int, long m, long n,
                                          float (&v)[8]) const {
        if (m >= p.M || n >= g.pitch) return;
        const int state = (int)rows[0];
        const float most = __uint_as_float(rows[0]), f = __uint_as_float(rows[1]);
        if (g.plane != 0) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = prod_exp((v[e] + l.bias[e] - most) * d.per) * f;
        } else {
            // (rounded to 16 bits next, by 2^-8 or 2^-11 of itself: the multiple's rounding, 2^-24 of the difference, is 2^-18 at q of e^-64)
            const float scale = 1.44269504f * d.per;
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = __builtin_amdgcn_exp2f((v[e] + l.bias[e] - most) * scale) * f;
        }
        // rows without entries, or with an entry that is none, and columns behind the last class
        if (row_odd(state) || n + 8 > p.N) {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = state == ROW_OUT || n + e >= p.N ? 0.f : state == ROW_BAD ? NAN : v[e];
        }
        operand_octet(g, m, n, g.pitch, v);
    }
};
// The same at the entries' places, from class `from` on, less their p.  Entries of one class are neighbours: the first writes for all.
__global__ __launch_bounds__(256) void distill_places_kernel(Kept kept, DistillGrad d, Out g, long rows, int k, long from, long n) {
    const long total = rows * k;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const int c = kept.classes[i];
        if (c < from || c >= from + n) continue;
        // (asked for together: a read's latency is most of this)
        const long m = i / k;
        const int j = (int)(i % k), before = j > 0 ? kept.classes[i - 1] : -1, after = j + 1 < k ? kept.classes[i + 1] : -1, state = kept.state[m];
        float p = kept.p[i];
        const float l = kept.at[i], sum = d.sum[m], f = d.factor(m);
        if (row_odd(state) || before == c) continue;
        if (after == c)
            for (int o = 1; j + o < k && kept.classes[i + o] == c; o++) p += kept.p[i + o];
        operand_one(g, m, c - from, (prod_exp((l - __int_as_float(state)) * d.per) / sum - p) * f);
    }
}

// ------------------------------------------------------------------------------------------------- on the host
struct DistillSizes : HeadSizes {
    int k, teacher;  // the teacher's type
    DistillSizes(size_t r, int c, int v, int entries, int t, int tt) : HeadSizes(r, c, v, t), k(entries), teacher(tt) {}
    bool ok() const { return HeadSizes::ok() && k >= 1 && k <= kDistillMost && known(teacher); }
};
// (T and 1 / T, their squares, and logits times either stay numbers of fp32 by far)
static bool temperature_ok(float T) { return T >= 1e-4f && T <= 1e4f; }

// Entries that are many of few classes: all logits are left, up to 256 MB of them, and the join takes those of the entries (forward, us, by the table of
// runs and this way: 4212 x 568 x 86, k = 81 in fp16 66, 33; 8192 x 512 x 4000, k = 200 in bf16 142, 106; 32768 x 256 x 150 in fp16 with k = 10 37, 32, 8 33,
// 30, 6 29.8, 28.7, but 5 28.3, 28.6; 8192 x 256 x 1000 with k = 32 31.8, 32.3)
static long logits_pitch(long V) { return (V + 3) / 4 * 4; }
static bool dense_entries(const DistillSizes &s) { return s.V <= 24 * (long)s.k && s.rows * logits_pitch(s.V) <= 1L << 26; }

static int distill_forward(const DistillSizes &s, const void *x, const void *w, const void *b, const void *logits, const long long *classes, float T,
                           float *keep, float *loss, float *count, bool mean, Arena &ws, hipStream_t st) {
    Staging stage;
    const Operand ox = stage.matrix(x, s.rows, s.C, s.dtype, ws), ow = stage.matrix(w, s.V, s.C, s.dtype, ws);
    int e = stage.launch(ws.dry(), st);
    if (e) return e;
    const Product p = make_product(ox, ow, s.rows, s.V, s.C, 0);
    const int width = wave_columns(tile_for(p.M, p.N, p.steps));
    const int parts = (int)((s.V + width - 1) / width);
    // (rows of a workgroup as in head_forward; few of many parts share them among more threads)
    const bool few = s.rows <= 128 && parts <= 256, narrow = !few && parts <= 16 && s.k <= 16;
    const int group = few || narrow ? 64 : 16;
    const int blocks = few ? 1 : (int)std::min((s.rows + group - 1) / group, 1L << 20);
    float2 *part = (float2 *)ws.take((size_t)parts * s.rows * sizeof(float2));
    const bool dense = dense_entries(s);
    const long wide = logits_pitch(s.V);
    unsigned *table = dense ? nullptr : (unsigned *)ws.take((size_t)s.rows * run_pitch(s.V) * sizeof(unsigned));
    float *all = dense ? (float *)ws.take((size_t)s.rows * wide * sizeof(float)) : nullptr;
    float2 *block = mean && blocks > 1 ? (float2 *)ws.take((size_t)blocks * sizeof(float2)) : nullptr;
    if (ws.dry()) return 0;
    const Kept kept(keep, s.rows, s.k);
    const float per = 1.f / T;
    auto *const entries = s.teacher == DWO_F32 ? launch_entries<float> : s.teacher == DWO_BF16 ? launch_entries<bf16_t> : launch_entries<f16_t>;
    if ((e = entries(logits, classes, kept, table, s.rows, s.V, s.k, per, st))) return e;
    const DistillStatsEpi epi{{b, s.dtype}, table, run_pitch(s.V), kept.classes, s.k, kept.at, all, part, 1.44269504f * per};
    if ((e = launch_product<false, false, false>(p, s.dtype, epi, st))) return e;
    const bool long_rows = !few && !narrow && parts >= 128;
    auto *const join = few ? distill_join_kernel<64, 16> : narrow ? distill_join_kernel<64, 4> : long_rows ? distill_join_kernel<16, 64> : distill_join_kernel<16, 16>;
    join<<<dim3((unsigned)blocks), dim3(few || long_rows ? 1024 : 256), 0, st>>>(part, kept, mean ? nullptr : loss, mean ? loss : nullptr, count, block, all, wide, s.rows,
                                                                                 parts, s.k, T);
    if (block != nullptr) head_mean_kernel<<<dim3(1), dim3(1024), 0, st>>>(block, blocks, loss, count);
    return status();
}

// Few rows and a large weight: dx has one tile and long sums, dw many tiles and short ones, and a tile that suits both takes longer than two launches (us of
// both passes together, and apart: fp32 17 x 296 x 47541 333, 244, 128 x 512 x 30000 315, 276; bf16 1 x 512 x 65536 167, 144, 64 rows 154, 153; but
// fp32 30 x 1024 x 10000 155, 162, 300 x 512 x 30000 402, 414)
static bool products_apart(const DistillSizes &s) { return s.rows <= 128 && s.V * s.C >= 12L << 20; }

static int distill_backward(const DistillSizes &s, const float *up, const void *x, const void *w, const void *b, const float *keep, float T,
                            const float *count, void *dx, void *dw, void *db, int grad, Arena &ws, hipStream_t st) {
    Staging stage;
    const Operand ox = stage.matrix(x, s.rows, s.C, s.dtype, ws), ow = stage.matrix(w, s.V, s.C, s.dtype, ws);
    int e = stage.launch(ws.dry(), st);
    if (e) return e;
    const Operand g = take_operand(ws, s.rows, up8(s.piece()), s.dtype, (double)s.rows * (double)s.C * (double)s.V);
    const bool mean = count != nullptr, half = s.dtype == DWO_F16;
    float *scale = half && !mean ? (float *)ws.take(2 * sizeof(float)) : nullptr;
    const Kept kept(const_cast<float *>(keep), s.rows, s.k);
    if (scale != nullptr && !ws.dry()) {
        head_scale_kernel<<<dim3(1), dim3(1024), 0, st>>>(up, RowStates{kept.state}, s.rows, scale);
        if ((e = status())) return e;
    }
    const DistillGrad d{kept.state, kept.sum, mean ? nullptr : up, scale, 1.f / T, half && mean ? kHalfScale : 1.f};
    auto make = [&](long from, long n, const Operand &wp, const Operand &gp) {
        const DistillGradEpi epi{{b != nullptr ? (const char *)b + from * size_of(s.dtype) : nullptr, s.dtype}, d, out_of(gp, s.dtype)};
        const int status_of = launch_product<false, false, false>(make_product(ox, wp, s.rows, n, s.C, 0), s.dtype, epi, st);
        if (status_of) return status_of;
        distill_places_kernel<<<dim3(blocks_for(s.rows * s.k, 8192)), dim3(256), 0, st>>>(kept, d, out_of(gp, s.dtype), s.rows, s.k, from, n);
        return status();
    };
    auto shared = [&](PlainEpi epi) {
        epi.alpha = mean ? up : scale != nullptr ? scale + 1 : nullptr;
        epi.over = count;
        epi.factor = T / (half && mean ? kHalfScale : 1.f);
        return epi;
    };
    return head_pieces(s, ox, ow, g, dx, dw, db, grad, make, shared, ws, st, products_apart(s));
}

}  // namespace dwo

using namespace dwo;

extern "C" {

size_t dwo_distill_workspace_bytes(size_t rows, int C, int V, int k, int backward, int dtype) {
    const DistillSizes s(rows, C, V, k, dtype, DWO_F32);
    if (!s.ok()) return 0;
    Arena ws = Arena::measure();
    void *const any = (void *)256;  // (nothing is launched)
    if (backward)
        distill_backward(s, (const float *)any, any, any, any, (const float *)any, 1.f, nullptr, any, any, any, DWO_F32, ws, nullptr);
    else
        distill_forward(s, any, any, any, any, (const long long *)any, 1.f, (float *)any, (float *)any, (float *)any, true, ws, nullptr);
    return ws.used + 256;
}

int dwo_distill_forward(const void *x, const void *w, const void *bias, const void *logits, const void *classes, float temperature, float *keep,
                        float *loss, float *count, void *ws, size_t ws_bytes, size_t rows, int C, int V, int k, int dtype, int logits_dtype,
                        void *stream) {
    if (!x || !w || !logits || !classes || !keep || !loss || !ws) return DWO_ERR_NULL_POINTER;
    if (!known(dtype) || !known(logits_dtype)) return DWO_ERR_BAD_DTYPE;
    const DistillSizes s(rows, C, V, k, dtype, logits_dtype);
    if (!s.ok() || !temperature_ok(temperature) || ((uintptr_t)x | (uintptr_t)w | (uintptr_t)ws) % 16 != 0 || (uintptr_t)classes % 8 != 0 ||
        (uintptr_t)keep % 4 != 0 || (uintptr_t)logits % size_of(logits_dtype) != 0)
        return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_distill_workspace_bytes(rows, C, V, k, 0, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    Arena a{(char *)ws, 0, ws_bytes};
    return distill_forward(s, x, w, bias, logits, (const long long *)classes, temperature, keep, loss, count, count != nullptr, a, (hipStream_t)stream);
}

int dwo_distill_backward(const float *up, const void *x, const void *w, const void *bias, const float *keep, float temperature, const float *count,
                         void *dx, void *dw, void *db, void *ws, size_t ws_bytes, size_t rows, int C, int V, int k, int dtype, int grad_dtype,
                         void *stream) {
    if (!up || !x || !w || !keep || !ws) return DWO_ERR_NULL_POINTER;
    if (!known(dtype) || !known(grad_dtype)) return DWO_ERR_BAD_DTYPE;
    const DistillSizes s(rows, C, V, k, dtype, DWO_F32);
    if (!s.ok() || !temperature_ok(temperature) || ((uintptr_t)x | (uintptr_t)w | (uintptr_t)ws) % 16 != 0 || (uintptr_t)keep % 4 != 0 || (db && !dw))
        return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_distill_workspace_bytes(rows, C, V, k, 1, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    Arena a{(char *)ws, 0, ws_bytes};
    return distill_backward(s, up, x, w, bias, keep, temperature, count, dx, dw, db, grad_dtype, a, (hipStream_t)stream);
}

}  // extern "C"
