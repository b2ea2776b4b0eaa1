// The k largest values of each row and their places, largest first, of equal ones the lowest place first; NaN is above everything, zeros are equal.
//
// A row is read once, into registers.  The k-th largest of the threads' own largest values is no more than the row's k-th largest: what is not
// below it are few, usually less than 2 k; they are gathered, sorted with their places, and the first k go out.  Where they are too many (rows of
// few distinct values, rows with NaN) the k-th largest is found by bisection over all values, and among the ones equal to it the last place
// that still counts.
#include <algorithm>

#include "dwo_product.h"

namespace dwo {

constexpr int kTopMost = 1024;  // k
typedef unsigned long long u64;

// Values as whole numbers in their order: sign and magnitude turned into two's complement, so that both zeros are 0 and values that are no
// number are beyond the infinities at either end.
template <typename T>
constexpr int kTopInf = sizeof(T) == 4 ? 0x7f800000 : std::is_same<T, f16_t>::value ? 0x7c00 : 0x7f80;
template <typename T>
__device__ __forceinline__ int top_order(unsigned bits) {
    constexpr unsigned TOP = sizeof(T) == 4 ? 0x80000000u : 0x8000u;
    const int sign = bits & TOP ? -1 : 0;
    return ((int)(bits & (TOP - 1)) ^ sign) - sign;
}
// the same with what is no number above everything, as a number without a sign: the bisections' order
template <typename T>
__device__ __forceinline__ unsigned top_key(unsigned bits) {
    const int s = top_order<T>(bits);
    return s > kTopInf<T> || s < -kTopInf<T> ? 0xffffffffu : (unsigned)s ^ 0x80000000u;
}
// larger is further in front: the key, then the lower place
__device__ __forceinline__ u64 top_entry(unsigned key, unsigned place) { return (u64)key << 32 | (0xffffffffu - place); }
__device__ __forceinline__ unsigned top_place(u64 entry) { return 0xffffffffu - (unsigned)entry; }

template <typename T>
__device__ __forceinline__ unsigned raw_bits(const T *p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const unsigned *>(p);
    else return *reinterpret_cast<const uint16_t *>(p);
}

// ------------------------------------------------------------------------------------------------- a wave a row
template <class F>
__device__ __forceinline__ unsigned wave_join(unsigned v, F &&f) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v = f(v, (unsigned)__shfl_xor((int)v, off, 64));
    return v;
}
__device__ __forceinline__ int lanes_below(u64 mask) {
    return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
}
// the largest v in (lo, hi] with count(v) >= k, or lo, which has it; or any below with no more than `enough`
template <class F>
__device__ __forceinline__ unsigned top_bisect(unsigned lo, unsigned hi, int k, int enough, F &&count) {
    while (lo < hi) {
        const unsigned mid = lo + (hi - lo) / 2 + 1;
        const int n = count(mid);
        if (n >= k) {
            lo = mid;
            if (n <= enough) break;
        } else {
            hi = mid - 1;
        }
    }
    return lo;
}

// Rows of up to 64 E values, k up to 64: place = lane + 64 e
constexpr int kWaveEntries = 128;
template <typename T, int E>
__global__ __launch_bounds__(256) void top_wave_kernel(const T *__restrict__ x, T *__restrict__ values, long long *__restrict__ places, long rows,
                                                       int V, int k) {
    __shared__ u64 entries[4][kWaveEntries];
    const int lane = threadIdx.x & 63;
    u64 *const mine = entries[threadIdx.x >> 6];
    for (long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (long)gridDim.x * 4) {
        const T *at = x + row * V;
        unsigned key[E], most = 0;  // (0: nothing, below all values)
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int c = lane + 64 * e;
            key[e] = c < V ? top_key<T>(raw_bits(at + c)) : 0u;
            most = max(most, key[e]);
        }
        const unsigned high = wave_join(most, [](unsigned a, unsigned b) { return max(a, b); });
        const unsigned low = wave_join(most, [](unsigned a, unsigned b) { return min(a, b); });
        const unsigned bound = max(top_bisect(low, high, k, k + k / 4 + 4, [&](unsigned v) { return (int)__popcll(__ballot(most >= v)); }), 1u);
        int n = 0;
        auto gather = [&](auto &&keep) {
            n = 0;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const bool in = keep(e, n);
                const u64 mask = __ballot(in);
                const int to = n + lanes_below(mask);
                if (in && to < kWaveEntries) mine[to] = top_entry(key[e], (unsigned)(lane + 64 * e));
                n += (int)__popcll(mask);
            }
        };
        gather([&](int e, int) { return key[e] >= bound; });
        if (n > kWaveEntries) {
            const unsigned last = max(top_bisect(bound, high, k, k, [&](unsigned v) {
                int c = 0;
#pragma unroll
                for (int e = 0; e < E; e++) c += (int)__popcll(__ballot(key[e] >= v));
                return c;
            }), 1u);
            int above = 0;
#pragma unroll
            for (int e = 0; e < E; e++) above += (int)__popcll(__ballot(key[e] > last));
            int equal = 0;  // places go up with e and then with the lane
            gather([&](int e, int) {
                const u64 same = __ballot(key[e] == last);
                const bool in = key[e] > last || (key[e] == last && equal + lanes_below(same) < k - above);
                equal += (int)__popcll(same);
                return in;
            });
        }
        // (a wave's writes to LDS are there for its reads, in order)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        // the place of each among them: how many are in front of it
        for (int i = lane; i < n; i += 64) {
            const u64 own = mine[i];
            int rank = 0;
            for (int j = 0; j < n; j++) rank += mine[j] > own ? 1 : 0;
            if (rank < k) {
                const unsigned c = top_place(own);
                values[row * k + rank] = at[c];
                places[row * k + rank] = (long long)c;
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ------------------------------------------------------------------------------------------------- a workgroup a row, or a part of one
// Largest first, n of them padded to a power of two with zeros
template <int THREADS>
__device__ __forceinline__ void top_sort(u64 *entries, int n) {
    int size = 2;
    while (size < n) size *= 2;
    for (int i = n + (int)threadIdx.x; i < size; i += THREADS) entries[i] = 0;
    __syncthreads();
    for (int run = 2; run <= size; run *= 2)
        for (int far = run / 2; far > 0; far /= 2) {
            for (int i = (int)threadIdx.x; i < size / 2; i += THREADS) {
                const int a = (i / far) * 2 * far + i % far, b = a + far;
                const u64 u = entries[a], v = entries[b];
                if ((u < v) == ((a & run) == 0)) entries[a] = v, entries[b] = u;
            }
            __syncthreads();
        }
}
// where a row's k go: values and places, or entries of a part for another launch
template <typename T>
struct TopOut {
    const T *x;  // the row
    T *values;
    long long *places;
    u64 *entries;
    __device__ __forceinline__ void put(int i, u64 entry) const {
        if (entries != nullptr) {
            entries[i] = entry;
            return;
        }
        const unsigned c = top_place(entry);
        values[i] = x[c];
        places[i] = (long long)c;
    }
};

template <typename T, int THREADS, int U>
struct TopSizes {
    static constexpr int kEntries = THREADS >= 1024 ? 4096 : 2048;
    static constexpr long kMost = (long)THREADS * 8 * U;  // values of a part that begins at a piece of eight; eight less elsewhere
};
// `parts` parts of `length` values a row
template <typename T, int THREADS, int U>
__global__ __launch_bounds__(THREADS) void top_kernel(const T *__restrict__ x, T *__restrict__ values, long long *__restrict__ places,
                                                      u64 *__restrict__ out, long rows, long V, int k, int parts, long length) {
    constexpr int WAVES = THREADS / 64, WORDS = 8 * sizeof(T) / 4, EACH = 4 / sizeof(T), CAP = TopSizes<T, THREADS, U>::kEntries;
    constexpr unsigned LOWEST = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, f16_t>::value ? 0xfc00fc00u : 0xff80ff80u;
    __shared__ u64 entries[CAP];
    __shared__ unsigned joined[2][WAVES], least[WAVES];
    __shared__ int number;
    const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
    const long total = rows * V;
    int turn = 0;
    // a sum over the workgroup, everywhere
    auto sum = [&](unsigned mine) {
        turn ^= 1;
        if (lane == 0) joined[turn][wave] = mine;
        __syncthreads();
        unsigned all = 0;
#pragma unroll
        for (int w = 0; w < WAVES; w++) all += joined[turn][w];
        return (int)all;
    };
    for (long job = blockIdx.x; job < rows * parts; job += gridDim.x) {
        const long row = job / parts, from = job % parts * length, size = min(length, V - from), begin = row * V + from;
        const long piece0 = begin / 8;
        const int lead = (int)(begin % 8), pieces = (int)((lead + size + 7) / 8);
        unsigned word[U][WORDS];
        // element e of a piece is value (u THREADS + thread) 8 + e - lead of the part
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int piece = u * THREADS + (int)threadIdx.x;
            const T *at = x + (piece0 + piece) * 8;
            if (piece < pieces && (piece0 + piece + 1) * 8 <= total) {
#pragma unroll
                for (int w = 0; w < WORDS / 4; w++) {
                    const mma_u4 q = reinterpret_cast<const mma_u4 *>(at)[w];
#pragma unroll
                    for (int i = 0; i < 4; i++) word[u][4 * w + i] = q[i];
                }
            } else {
#pragma unroll
                for (int w = 0; w < WORDS; w++) word[u][w] = LOWEST;
            }
        }
        auto set = [&](unsigned &w, int half, unsigned bits) {
            if constexpr (EACH == 1) w = bits;
            else w = half ? (w & 0xffffu) | bits << 16 : (w & 0xffff0000u) | (bits & 0xffffu);
        };
        // pieces that hold values of other rows, and one that the tensor ends in
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int piece = u * THREADS + (int)threadIdx.x;
            const long first = (long)piece * 8 - lead;
            if (piece < pieces && (first < 0 || first + 8 > size)) {
                const bool read = (piece0 + piece + 1) * 8 <= total;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const long i = first + e;
                    if (i < 0 || i >= size) set(word[u][e / EACH], e % EACH, LOWEST);
                    else if (!read) set(word[u][e / EACH], e % EACH, raw_bits(x + begin + i));
                }
            }
        }
        int high = -kTopInf<T>, low = kTopInf<T>;
        if constexpr (EACH == 1) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int w = 0; w < WORDS; w++) {
                    const int s = top_order<T>(word[u][w]);
                    high = max(high, s), low = min(low, s);
                }
        } else {
            typedef short two __attribute__((ext_vector_type(2)));
            two most = {(short)high, (short)high}, fewest = {(short)low, (short)low};
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int w = 0; w < WORDS; w++) {
                    const two v = __builtin_bit_cast(two, word[u][w]), sign = v >> 15;
                    const two s = ((v & (short)0x7fff) ^ sign) - sign;
                    most = __builtin_elementwise_max(most, s), fewest = __builtin_elementwise_min(fewest, s);
                }
            high = max((int)most[0], (int)most[1]), low = min((int)fewest[0], (int)fewest[1]);
        }
        auto element = [&](int u, int e) {
            const unsigned w = word[u][e / EACH];
            return top_key<T>(EACH == 1 ? w : e % 2 ? w >> 16 : w & 0xffffu);
        };
        auto place = [&](int u, int e) { return (u * THREADS + (int)threadIdx.x) * 8 + e - lead; };
        const bool odd = high > kTopInf<T> || low < -kTopInf<T>;
        const unsigned own = (unsigned)high ^ 0x80000000u;
        const unsigned top = wave_join(own, [](unsigned a, unsigned b) { return max(a, b); });
        const unsigned bottom = wave_join(own, [](unsigned a, unsigned b) { return min(a, b); });
        __syncthreads();  // (the last row's entries are read)
        if (lane == 0) least[wave] = bottom;
        if (threadIdx.x == 0) number = 0;
        turn ^= 1;
        if (lane == 0) joined[turn][wave] = top;
        bool hard = __syncthreads_or(odd) != 0;
        unsigned hi = 0, lo = 0xffffffffu;
#pragma unroll
        for (int w = 0; w < WAVES; w++) hi = max(hi, joined[turn][w]), lo = min(lo, least[w]);
        constexpr unsigned NONE = (unsigned)(-kTopInf<T>) ^ 0x80000000u;
        const int want = (int)min((long)k, size);
        if (!hard) {
            const unsigned bound = want > THREADS ? NONE : top_bisect(lo, hi, want, want + want / 4 + 16, [&](unsigned v) { return sum((unsigned)__popcll(__ballot(own >= v))); });
            if (own >= bound)
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const unsigned key = element(u, e);
                        const int i = place(u, e);
                        if (key >= bound && i >= 0 && i < (int)size) {
                            const int to = atomicAdd(&number, 1);
                            if (to < CAP) entries[to] = top_entry(key, (unsigned)(from + i));
                        }
                    }
            __syncthreads();
            hard = number > CAP;
        }
        int n = number;
        if (hard) {
            // (rare: the values again from memory, each time, so that their keys and places take no registers from the others)
            const T *const part = x + begin;
            auto count = [&](auto &&in) {
                unsigned c = 0;
#pragma unroll 1
                for (int i = (int)threadIdx.x; i < (int)size; i += THREADS) c += in(top_key<T>(raw_bits(part + i)), i) ? 1 : 0;
                return sum(wave_join(c, [](unsigned a, unsigned b) { return a + b; }));
            };
            const unsigned last = top_bisect(NONE, 0xffffffffu, want, want, [&](unsigned v) { return count([&](unsigned key, int) { return key >= v; }); });
            const int rest = want - count([&](unsigned key, int) { return key > last; });
            // (the least place with `rest` equal ones up to it)
            int a = 0, b = (int)size - 1;
            while (a < b) {
                const int mid = a + (b - a) / 2;
                if (count([&](unsigned key, int i) { return key == last && i <= mid; }) >= rest) b = mid;
                else a = mid + 1;
            }
            __syncthreads();
            if (threadIdx.x == 0) number = 0;
            __syncthreads();
#pragma unroll 1
            for (int i = (int)threadIdx.x; i < (int)size; i += THREADS) {
                const unsigned key = top_key<T>(raw_bits(part + i));
                if (key > last || (key == last && i <= a)) entries[atomicAdd(&number, 1)] = top_entry(key, (unsigned)(from + i));
            }
            __syncthreads();
            n = number;
        }
        top_sort<THREADS>(entries, n);
        const TopOut<T> to = {x + row * V, out != nullptr ? nullptr : values + row * k, out != nullptr ? nullptr : places + row * k,
                              out != nullptr ? out + job * k : nullptr};
        for (int i = (int)threadIdx.x; i < k; i += THREADS)
            if (i < want) to.put(i, entries[i]);
            else if (out != nullptr) out[job * k + i] = 0;  // (a part of fewer values: nothing)
    }
}

// Entries of `parts` parts joined, `group` parts a workgroup, until one is left
constexpr int kJoinEntries = 4096;
template <typename T>
__global__ __launch_bounds__(1024) void top_join_kernel(const u64 *__restrict__ in, const T *__restrict__ x, T *__restrict__ values,
                                                        long long *__restrict__ places, u64 *__restrict__ out, long rows, long V, int k, int parts,
                                                        int group) {
    __shared__ u64 entries[kJoinEntries];
    const int after = (parts + group - 1) / group;
    for (long job = blockIdx.x; job < rows * after; job += gridDim.x) {
        const long row = job / after;
        const int part = (int)(job % after) * group, n = min(group, parts - part) * k;
        __syncthreads();
        for (int i = (int)threadIdx.x; i < n; i += 1024) entries[i] = in[(row * parts + part) * k + i];
        top_sort<1024>(entries, n);
        const TopOut<T> to = {x + row * V, out != nullptr ? nullptr : values + row * k, out != nullptr ? nullptr : places + row * k,
                              out != nullptr ? out + job * k : nullptr};
        for (int i = (int)threadIdx.x; i < k; i += 1024) to.put(i, entries[i]);
    }
}

struct TopPlan {
    long rows, V;
    int k, dtype;
    bool ok() const {
        return rows >= 1 && rows <= 1L << 30 && V >= 1 && V <= 1L << 24 && k >= 1 && k <= kTopMost && k <= V && rows <= (1L << 40) / V && known(dtype);
    }
    bool wave() const { return V <= 1024 && k <= 64; }
    bool small() const { return V <= TopSizes<float, 256, 8>::kMost - 8; }
    int parts() const {
        const long most = TopSizes<float, 1024, 8>::kMost - (V % 8 == 0 ? 0 : 8);
        return wave() || small() ? 1 : (int)((V + most - 1) / most);
    }
    long length() const { return ((V + parts() - 1) / parts() + 7) / 8 * 8; }
    static int after(int parts, int k) { return (parts + kJoinEntries / k - 1) / (kJoinEntries / k); }
};
static unsigned top_blocks(long n) { return (unsigned)std::min(n, 1L << 20); }
template <typename T>
static int top_typed(const TopPlan &p, const T *x, T *values, long long *places, Arena &ws, hipStream_t st) {
    if (p.wave()) {
        if (ws.dry()) return 0;
        auto *kernel = p.V <= 256 ? top_wave_kernel<T, 4> : top_wave_kernel<T, 16>;
        kernel<<<dim3(top_blocks((p.rows + 3) / 4)), dim3(256), 0, st>>>(x, values, places, p.rows, (int)p.V, p.k);
        return status();
    }
    int parts = p.parts();
    const size_t room = (size_t)p.rows * parts * p.k * sizeof(u64);
    u64 *in = parts > 1 ? (u64 *)ws.take(room) : nullptr, *out = parts > 1 ? (u64 *)ws.take(room) : nullptr;
    if (ws.dry()) return 0;
    const long length = parts > 1 ? p.length() : p.V;
    if (p.small())
        top_kernel<T, 256, 8><<<dim3(top_blocks(p.rows)), dim3(256), 0, st>>>(x, values, places, in, p.rows, p.V, p.k, 1, length);
    else
        top_kernel<T, 1024, 8><<<dim3(top_blocks(p.rows * parts)), dim3(1024), 0, st>>>(x, values, places, in, p.rows, p.V, p.k, parts, length);
    int e = status();
    while (parts > 1 && e == 0) {
        const int group = kJoinEntries / p.k, after = TopPlan::after(parts, p.k);
        top_join_kernel<T><<<dim3(top_blocks(p.rows * after)), dim3(1024), 0, st>>>(in, x, values, places, after > 1 ? out : nullptr, p.rows, p.V, p.k,
                                                                                    parts, group);
        e = status();
        std::swap(in, out);
        parts = after;
    }
    return e;
}
static int top_run(const TopPlan &p, const void *x, void *values, long long *places, Arena &ws, hipStream_t st) {
    if (p.dtype == DWO_F32) return top_typed(p, (const float *)x, (float *)values, places, ws, st);
    if (p.dtype == DWO_BF16) return top_typed(p, (const bf16_t *)x, (bf16_t *)values, places, ws, st);
    return top_typed(p, (const f16_t *)x, (f16_t *)values, places, ws, st);
}

}  // namespace dwo

using namespace dwo;

extern "C" {

size_t dwo_top_workspace_bytes(size_t rows, int V, int k, int dtype) {
    const TopPlan p{(long)rows, V, k, dtype};
    if (!p.ok()) return 0;
    Arena ws = Arena::measure();
    top_run(p, nullptr, nullptr, nullptr, ws, nullptr);
    return ws.used + 256;
}

int dwo_top(const void *x, void *values, void *places, void *ws, size_t ws_bytes, size_t rows, int V, int k, int dtype, void *stream) {
    if (!x || !values || !places || !ws) return DWO_ERR_NULL_POINTER;
    if (!known(dtype)) return DWO_ERR_BAD_DTYPE;
    const TopPlan p{(long)rows, V, k, dtype};
    if (!p.ok() || ((uintptr_t)x | (uintptr_t)ws) % 16 != 0 || (uintptr_t)places % 8 != 0 || (uintptr_t)values % size_of(dtype) != 0)
        return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_top_workspace_bytes(rows, V, k, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    Arena a{(char *)ws, 0, ws_bytes};
    return top_run(p, x, values, (long long *)places, a, (hipStream_t)stream);
}

}  // extern "C"
