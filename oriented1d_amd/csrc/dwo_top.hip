// The k largest values of each row and their places, largest first, of equal ones the lowest place first; NaN is above everything, zeros are equal.
//
// A row is read once for the largest values of its units, a few neighbouring pieces each.  The k-th largest of these is no more than the row's k-th
// largest; it is found by bisection, and need not be met exactly.  Only units that reach it can hold one of the k: little more than k of two thousand.
// They are read again, what reaches the bound is gathered, usually less than 3/2 k, and each entry's place among the others is the number in front of
// it.  Where too many are gathered (rows of few distinct values, or of fewer than k finite ones among -infinity) the k-th largest itself is found by bisection
// over all values, and among those equal to it the last place that still counts (8192 rows of 65536, k = 64, bf16: zeros 2.9 ms, 32 finite values among
// -infinity 5.0, a NaN with a sign in each 6.3, in fp32 6.2, 16 and 13; 0.2 and 0.37 of any values).
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
// the same with what is no number above everything, one key for all of them, as a number without a sign: the bisections' order
template <typename T>
__device__ __forceinline__ unsigned order_key(int s) {
    return s > kTopInf<T> || s < -kTopInf<T> ? 0xffffffffu : (unsigned)s ^ 0x80000000u;
}
template <typename T>
__device__ __forceinline__ unsigned top_key(unsigned bits) { return order_key<T>(top_order<T>(bits)); }
// the value of a key; of zeros and of what is no number it is in memory
template <typename T>
__device__ __forceinline__ T key_value(unsigned key) {
    const unsigned s = key ^ 0x80000000u, sign = s & 0x80000000u, magnitude = sign != 0 ? 0u - s : s;
    if constexpr (sizeof(T) == 4) return __uint_as_float(sign | magnitude);
    else return __builtin_bit_cast(T, (uint16_t)(sign >> 16 | magnitude));
}
template <typename T>
__device__ __forceinline__ T top_value(unsigned key, const T *at) {
    return key == 0x80000000u || key == 0xffffffffu ? *at : key_value<T>(key);
}
// larger is further in front: the key, then the lower place
__device__ __forceinline__ u64 top_entry(unsigned key, unsigned place) { return (u64)key << 32 | (0xffffffffu - place); }
__device__ __forceinline__ unsigned top_place(u64 entry) { return 0xffffffffu - (unsigned)entry; }

template <typename T>
__device__ __forceinline__ unsigned raw_bits(const T *p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const unsigned *>(p);
    else return *reinterpret_cast<const uint16_t *>(p);
}

template <int CTRL>
__device__ __forceinline__ unsigned top_dpp(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
// over G neighbouring lanes (16, 32 or 64), in every one of them
template <int G, class F>
__device__ __forceinline__ unsigned lanes_join(unsigned v, F &&f) {
    v = f(v, top_dpp<0xB1>(v));   // quad_perm [1,0,3,2]
    v = f(v, top_dpp<0x4E>(v));   // quad_perm [2,3,0,1]
    v = f(v, top_dpp<0x141>(v));  // row_half_mirror
    v = f(v, top_dpp<0x140>(v));  // row_mirror
    if constexpr (G >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = f((unsigned)s[0], (unsigned)s[1]);
    }
    if constexpr (G >= 64) {
        const auto t = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = f((unsigned)t[0], (unsigned)t[1]);
    }
    return v;
}
struct Larger {
    __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return max(a, b); }
};
struct Smaller {
    __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return min(a, b); }
};
struct Total {
    __device__ __forceinline__ unsigned operator()(unsigned a, unsigned b) const { return a + b; }
};
__device__ __forceinline__ int lanes_below(u64 mask) {
    return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
}
// The largest v in (lo, hi] with count(v) >= k, or lo, which has it; or one below with no more than `enough`.  Every other step goes to the middle of
// the values, which the k-th largest is near to where values are spread as usual (of fp32 logits half a dozen steps, where the middle of keys, through
// all the exponents, takes some twenty); the steps between end it in any case.
template <typename T, class F>
__device__ __forceinline__ unsigned top_bisect(unsigned lo, unsigned hi, int k, int enough, F &&count) {
    for (bool by_value = true; lo < hi; by_value = !by_value) {
        unsigned mid = lo + (hi - lo) / 2 + 1;
        if (by_value) {
            const T v = from_float<T>(0.5f * to_float(key_value<T>(lo)) + 0.5f * to_float(key_value<T>(hi)));
            const unsigned key = top_key<T>(raw_bits(&v));
            mid = key > lo && key <= hi ? key : mid;
        }
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
__device__ __forceinline__ int top_enough(int k) { return k + k / 4 + 8; }
// of those that are gathered: what is sorted is a power of two
__device__ __forceinline__ int top_enough_entries(int k) { return min(top_enough(k), k > 1 ? 1 << (32 - __builtin_clz(k - 1)) : 1); }
__device__ __forceinline__ int top_refined(int k) { return max(256, k + k / 2); }

// ------------------------------------------------------------------------------------------------- short rows
// Rows of up to G E values, G lanes each and k up to G: place = lane + G e; the lanes are the units.  The 64 / G rows of a wave go through the same
// steps, each lane with its own row's numbers.
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void top_lanes_kernel(const T *__restrict__ x, T *__restrict__ values, long long *__restrict__ places, long rows,
                                                        int V, int k) {
    constexpr int ROWS = 256 / G, CAP = 2 * G;  // entries of a row
    typedef std::conditional_t<G == 64, u64, unsigned> Mask;
    // (rows 16 bytes apart in their banks: each wave reads one place of all its rows at a time)
    __shared__ __attribute__((aligned(16))) u64 entries[ROWS][CAP + 2];
    const int lane = threadIdx.x % G;
    const bool upper = (threadIdx.x & 32) != 0;
    const int shift = G == 16 ? threadIdx.x & 16 : 0;
    u64 *const mine = entries[threadIdx.x / G];
    // those of the row's lanes for which it is true, and how many
    auto those = [&](bool in) -> Mask {
        const u64 all = __ballot(in);
        if constexpr (G == 64) {
            return all;
        } else {
            const unsigned half = upper ? (unsigned)(all >> 32) : (unsigned)all;
            return G == 32 ? half : half >> shift & 0xffffu;
        }
    };
    auto number = [](Mask m) { return G == 64 ? (int)__popcll((u64)m) : __popc((unsigned)m); };
    const Mask below = ((Mask)1 << lane) - 1;
    for (long first = (long)blockIdx.x * ROWS; first < rows; first += (long)gridDim.x * ROWS) {
        const long row = first + threadIdx.x / G;
        const bool real = row < rows;
        const T *const base = x + first * V;  // (of the workgroup)
        const unsigned at = (unsigned)((threadIdx.x / G) * V + lane);
        unsigned key[E], most = 0;  // (0: nothing, below all values)
#pragma unroll
        for (int e = 0; e < E; e++) key[e] = real && lane + G * e < V ? raw_bits(base + at + G * e) : ~0u;
#pragma unroll
        for (int e = 0; e < E; e++) key[e] = lane + G * e < V && real ? top_key<T>(key[e]) : 0u;
#pragma unroll
        for (int e = 0; e < E; e++) most = max(most, key[e]);
        const unsigned high = lanes_join<G>(most, Larger{}), low = lanes_join<G>(most, Smaller{});
        unsigned bound = max(top_bisect<T>(low, high, k, k + k / 4 + 1, [&](unsigned v) { return number(those(most >= v)); }), 1u);
        // how many of the lane's, and of the row's in all; a lane's go behind those of the lanes below it
        int own = 0;
#pragma unroll
        for (int e = 0; e < E; e++) own += key[e] >= bound ? 1 : 0;
        int n = (int)lanes_join<G>((unsigned)own, Total{});
        if (__any(n > CAP)) {
            bound = max(top_bisect<T>(bound, high, k, k, [&](unsigned v) {
                int c = 0;
#pragma unroll
                for (int e = 0; e < E; e++) c += number(those(key[e] >= v));
                return c;
            }), 1u);
            int rest = k, equal = 0;
#pragma unroll
            for (int e = 0; e < E; e++) rest -= number(those(key[e] > bound));
            // (places go up with e and then with the lane)
            own = 0;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const Mask same = those(key[e] == bound);
                const bool in = key[e] > bound || (key[e] == bound && equal + number(same & below) < rest);
                equal += number(same);
                if (!in) key[e] = 0;
                own += in ? 1 : 0;
            }
            n = (int)lanes_join<G>((unsigned)own, Total{});
        }
        int to = 0;  // the number of entries of the lanes below: a bit of it at a time
#pragma unroll
        for (int bit = 0; (1 << bit) <= E; bit++) to += number(those((own >> bit & 1) != 0) & below) << bit;
#pragma unroll
        for (int e = 0; e < E; e++)
            if (key[e] >= bound) mine[to++] = top_entry(key[e], (unsigned)(lane + G * e));
        if (lane == 0) mine[n] = 0;  // (two are read at a time)
        // (a wave's writes to LDS are there for its reads, in order)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        // two entries a lane at the most, each one's place the number in front of it
        const u64 entry[2] = {lane < n ? mine[lane] : 0, lane + G < n ? mine[lane + G] : 0};
        int rank[2] = {};
        for (int j = 0; j < n; j += 2) {
            typedef u64 two __attribute__((ext_vector_type(2)));
            const two other = *reinterpret_cast<const two *>(mine + j);
#pragma unroll
            for (int h = 0; h < 2; h++) rank[h] += (other[0] > entry[h] ? 1 : 0) + (other[1] > entry[h] ? 1 : 0);
        }
        if (real)
#pragma unroll
            for (int h = 0; h < 2; h++)
                if (lane + h * G < n && rank[h] < k) {
                    const unsigned c = top_place(entry[h]);
                    values[row * k + rank[h]] = top_value((unsigned)(entry[h] >> 32), x + row * V + c);
                    places[row * k + rank[h]] = (long long)c;
                }
        __builtin_amdgcn_wave_barrier();
    }
}

// ------------------------------------------------------------------------------------------------- a workgroup a row, or a part of one
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
        values[i] = top_value((unsigned)(entry >> 32), x + c);
        places[i] = (long long)c;
    }
};
// The first `want` of n entries, in order.  Up to 256: each entry's place is the number in front of it, counted by neighbouring lanes together; above, they
// are sorted (8192 rows of 16384, k = 200, some 270 entries: 147 us, counted 158; 4096 rows of 32768, k = 120: 73 us, from 128 on sorted 85).
template <int THREADS, class Out>
__device__ __forceinline__ void top_order_out(u64 *entries, int n, int want, const Out &out) {
    int size = 2;
    while (size < n) size *= 2;
    if (size <= (THREADS < 256 ? THREADS : 256)) {
        const int share = min(THREADS / size, 8), i = (int)threadIdx.x / share, part = (int)threadIdx.x % share;
        const u64 own = i < n ? entries[i] : 0;
        int rank = 0;
        if (i < n)
#pragma unroll 4
            for (int j = part; j < n; j += share) rank += entries[j] > own ? 1 : 0;
        for (int off = 1; off < share; off *= 2) rank += __shfl_xor(rank, off, 64);
        if (i < n && part == 0 && rank < want) out.put(rank, own);
        return;
    }
    if (THREADS == 128 && size == 256) {
        const int i = (int)threadIdx.x, k = i + THREADS;
        const u64 own[2] = {entries[i], k < n ? entries[k] : 0};  // (more than 128 are there)
        int rank[2] = {};
#pragma unroll 4
        for (int j = 0; j < n; j++) {
            const u64 other = entries[j];
            rank[0] += other > own[0] ? 1 : 0, rank[1] += other > own[1] ? 1 : 0;
        }
        if (rank[0] < want) out.put(rank[0], own[0]);
        if (k < n && rank[1] < want) out.put(rank[1], own[1]);
        return;
    }
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
    for (int i = (int)threadIdx.x; i < want; i += THREADS) out.put(i, entries[i]);
}

// Eight values in a lane's registers: their order's extremes, and each one's key
template <typename T>
struct TopPiece {
    static constexpr int WORDS = 2 * sizeof(T);
    unsigned word[WORDS];
    __device__ __forceinline__ void read(const T *at) {
#pragma unroll
        for (int w = 0; w < WORDS / 4; w++) {
            const mma_u4 q = reinterpret_cast<const mma_u4 *>(at)[w];
#pragma unroll
            for (int i = 0; i < 4; i++) word[4 * w + i] = q[i];
        }
    }
    __device__ __forceinline__ unsigned key(int e) const {
        if constexpr (sizeof(T) == 4) return top_key<T>(word[e]);
        else return top_key<T>(e % 2 ? word[e / 2] >> 16 : word[e / 2] & 0xffffu);
    }
};
template <typename T>
struct TopRange {  // largest and smallest order so far: of halves of words for 16 bits
    typedef std::conditional_t<sizeof(T) == 4, int, short __attribute__((ext_vector_type(2)))> V;
    V most, least;
    __device__ __forceinline__ TopRange() {
        constexpr int I = kTopInf<T>;
        if constexpr (sizeof(T) == 4) most = -I, least = I;
        else most = V{(short)-I, (short)-I}, least = V{(short)I, (short)I};
    }
    __device__ __forceinline__ void meet(const TopPiece<T> &p) {
#pragma unroll
        for (int w = 0; w < TopPiece<T>::WORDS; w++) {
            if constexpr (sizeof(T) == 4) {
                const int s = top_order<T>(p.word[w]);
                most = max(most, s), least = min(least, s);
            } else {
                const V v = __builtin_bit_cast(V, p.word[w]), sign = v >> 15;
                const V s = ((v & (short)0x7fff) ^ sign) - sign;
                most = __builtin_elementwise_max(most, s), least = __builtin_elementwise_min(least, s);
            }
        }
    }
    __device__ __forceinline__ int high() const {
        if constexpr (sizeof(T) == 4) return most;
        else return max((int)most[0], (int)most[1]);
    }
    __device__ __forceinline__ int low() const {
        if constexpr (sizeof(T) == 4) return least;
        else return min((int)least[0], (int)least[1]);
    }
};

constexpr int kTopUnits = 4;  // of a thread: pieces u of it with u % 4 alike
template <int THREADS>
constexpr int kTopEntries = THREADS >= 512 ? 4096 : 2048;
// `parts` parts of `length` values a row
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS < 512 ? 4 : sizeof(T) == 4 ? 6 : 8) void top_kernel(const T *__restrict__ x, T *__restrict__ values, long long *__restrict__ places,
                                                      u64 *__restrict__ out, long rows, long V, int k, int parts, long length) {
    constexpr int WAVES = THREADS / 64, UNITS = kTopUnits, CAP = kTopEntries<THREADS>;  // (k is at most four times THREADS, as units are)
    constexpr unsigned NONE = (unsigned)(-kTopInf<T>) ^ 0x80000000u;
    __shared__ u64 entries[CAP];
    __shared__ uint16_t hot[THREADS * UNITS];
    __shared__ unsigned joined[2][WAVES], least[WAVES];
    __shared__ int number, units;
    const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
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
        const long row = job / parts, from = job % parts * length, begin = row * V + from;
        const int size = (int)min(length, V - from), lead = (int)(begin % 8), want = min(k, size);
        // whole pieces lie from `inner` on, q of them behind `skip` values; the values in front and behind go one to a thread
        const int skip = min((8 - lead) % 8, size), q = (size - skip) / 8, behind = skip + 8 * q;
        const T *const part = x + begin, *const inner = part + skip;
        const int edge = (int)threadIdx.x < skip ? (int)threadIdx.x : behind + (int)threadIdx.x - skip;  // (of the first threads)
        const unsigned edge_key = edge < size && (int)threadIdx.x < 16 ? top_key<T>(raw_bits(part + edge)) : 0u;
        unsigned own[UNITS];
        TopRange<T> all;
        {
            TopRange<T> range[UNITS];
            // (one piece of each unit on its way: with two of 16 bits the registers of two thousand threads a CU do not suffice, 222 us and 72 MB of spills)
            for (int p = (int)threadIdx.x; p < q; p += UNITS * THREADS) {
                TopPiece<T> piece[UNITS];
#pragma unroll
                for (int u = 0; u < UNITS; u++)
                    if (p + u * THREADS < q) piece[u].read(inner + 8L * (p + u * THREADS));
#pragma unroll
                for (int u = 0; u < UNITS; u++)
                    if (p + u * THREADS < q) range[u].meet(piece[u]);
            }
            int low = kTopInf<T>, high = -kTopInf<T>;
#pragma unroll
            for (int u = 0; u < UNITS; u++) {
                high = max(high, range[u].high()), low = min(low, range[u].low());
                own[u] = order_key<T>(range[u].high());  // (never below -infinity)
            }
            // (what is no number and has no sign is above the infinities there too; with a sign it is below everything, and its unit may be missed)
            const bool odd = low < -kTopInf<T>;
            unsigned bottom = 0xffffffffu;  // of units with a piece
#pragma unroll
            for (int u = 0; u < UNITS; u++) bottom = min(bottom, (int)threadIdx.x + u * THREADS < q ? own[u] : 0xffffffffu);
            const unsigned top = lanes_join<64>(max(order_key<T>(high), edge_key), Larger{});
            bottom = lanes_join<64>(bottom, Smaller{});
            __syncthreads();  // (what the last row left is read)
            turn ^= 1;
            if (lane == 0) joined[turn][wave] = top, least[wave] = bottom;
            if (threadIdx.x == 0) number = 0, units = 0;
            if (__syncthreads_or(odd)) own[0] = 0;  // (below every value: marks such a row)
        }
        bool hard = own[0] == 0;
        unsigned least_last = NONE, most_last = 0xffffffffu;  // between which the k-th largest is
        if (!hard) {
            unsigned hi = 0, lo = 0xffffffffu;
#pragma unroll
            for (int w = 0; w < WAVES; w++) hi = max(hi, joined[turn][w]), lo = min(lo, least[w]);
            // (too few units: every value is gathered)
            const unsigned bound = q < want ? NONE : top_bisect<T>(lo, hi, want, top_enough(want), [&](unsigned v) {
                unsigned c = 0;
#pragma unroll
                for (int u = 0; u < UNITS; u++) c += (unsigned)__popcll(__ballot(own[u] >= v));
                return sum(c);
            });
            auto keep = [&](unsigned key, int i) {
                const int to = atomicAdd(&number, 1);
                if (to < CAP) entries[to] = top_entry(key, (unsigned)(from + i));
            };
#pragma unroll
            for (int u = 0; u < UNITS; u++)
                if (own[u] >= bound) hot[atomicAdd(&units, 1)] = (uint16_t)(u * THREADS + (int)threadIdx.x);
            if (edge_key >= bound) keep(edge_key, edge);
            __syncthreads();
            // pieces of a unit, rounded up to a power of two, one a thread
            const int each = (q + UNITS * THREADS - 1) / (UNITS * THREADS), log = each > 1 ? 32 - __builtin_clz(each - 1) : 0, tasks = units << log;
            for (int t = (int)threadIdx.x; t < tasks; t += THREADS) {
                const int p = (t & ((1 << log) - 1)) * UNITS * THREADS + hot[t >> log];
                if (p >= q) continue;
                TopPiece<T> piece;
                piece.read(inner + 8L * p);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const unsigned key = piece.key(e);
                    if (key >= bound) keep(key, skip + 8 * p + e);
                }
            }
            __syncthreads();
            hard = number > CAP;
            least_last = bound, most_last = hi > ((unsigned)kTopInf<T> ^ 0x80000000u) ? 0xffffffffu : hi;
        }
        int n = number;
        if (!hard && n > top_refined(want)) {
            // few units for so many: the bound lets many through, and the k-th largest is looked for among them
            const unsigned last = top_bisect<T>(least_last, most_last, want, top_enough_entries(want), [&](unsigned v) {
                unsigned c = 0;
                for (int i = (int)threadIdx.x; i < n; i += THREADS) c += (unsigned)(entries[i] >> 32) >= v ? 1u : 0u;
                return sum(lanes_join<64>(c, Total{}));
            });
            __syncthreads();
            if (threadIdx.x == 0) number = 0;
            // (what stays goes to places that have been read)
            for (int first = 0; first < n; first += THREADS) {
                const int i = first + (int)threadIdx.x;
                const u64 entry = i < n ? entries[i] : 0;
                __syncthreads();
                if (i < n && (unsigned)(entry >> 32) >= last) entries[atomicAdd(&number, 1)] = entry;
            }
            __syncthreads();
            n = number;
        }
        if (hard) {
            // (rare: all values again from memory, each time)
            auto visit = [&](auto &&f) {
                if (edge_key != 0) f(edge_key, edge);
#pragma unroll 1
                for (int p = (int)threadIdx.x; p < q; p += THREADS) {
                    TopPiece<T> piece;
                    piece.read(inner + 8L * p);
#pragma unroll
                    for (int e = 0; e < 8; e++) f(piece.key(e), skip + 8 * p + e);
                }
            };
            auto count = [&](auto &&in) {
                unsigned c = 0;
                visit([&](unsigned key, int i) { c += in(key, i) ? 1 : 0; });
                return sum(lanes_join<64>(c, Total{}));
            };
            const unsigned last = top_bisect<T>(least_last, most_last, want, want, [&](unsigned v) { return count([&](unsigned key, int) { return key >= v; }); });
            const int rest = want - count([&](unsigned key, int) { return key > last; });
            // (the least place with `rest` equal ones up to it)
            int a = 0, b = size - 1;
            while (a < b) {
                const int mid = a + (b - a) / 2;
                if (count([&](unsigned key, int i) { return key == last && i <= mid; }) >= rest) b = mid;
                else a = mid + 1;
            }
            __syncthreads();
            if (threadIdx.x == 0) number = 0;
            __syncthreads();
            visit([&](unsigned key, int i) {
                if (key > last || (key == last && i <= a)) entries[atomicAdd(&number, 1)] = top_entry(key, (unsigned)(from + i));
            });
            __syncthreads();
            n = number;
        }
        const TopOut<T> to = {x + row * V, out != nullptr ? nullptr : values + row * k, out != nullptr ? nullptr : places + row * k,
                              out != nullptr ? out + job * k : nullptr};
        top_order_out<THREADS>(entries, n, want, to);
        if (out != nullptr)
            for (int i = want + (int)threadIdx.x; i < k; i += THREADS) out[job * k + i] = 0;  // (a part of fewer values: nothing)
    }
}

// Entries of `parts` parts joined, `group` parts a workgroup, until one is left.  Each part's are in order: with each part's first ceil(k / parts), k
// entries or more are no less than the least of these parts' last ones, which few others reach.
constexpr int kJoinEntries = 4096;
template <typename T>
__global__ __launch_bounds__(512) void top_join_kernel(const u64 *__restrict__ in, const T *__restrict__ x, T *__restrict__ values,
                                                       long long *__restrict__ places, u64 *__restrict__ out, long rows, long V, int k, int parts,
                                                       int group) {
    __shared__ u64 entries[kJoinEntries];
    __shared__ unsigned low[8];
    __shared__ int number;
    const int after = (parts + group - 1) / group;
    for (long job = blockIdx.x; job < rows * after; job += gridDim.x) {
        const long row = job / after;
        const int part = (int)(job % after) * group, count = min(group, parts - part), n = count * k;
        const u64 *const from = in + (row * parts + part) * k;
        constexpr int EACH = kJoinEntries / 512;
        u64 held[EACH];
        const int first = (k + count - 1) / count;
        unsigned last = 0xffffffffu;
        for (int i = (int)threadIdx.x; i < count; i += 512) last = min(last, (unsigned)(from[(long)i * k + first - 1] >> 32));
#pragma unroll
        for (int u = 0; u < EACH; u++) {
            const int i = (int)threadIdx.x + 512 * u;
            held[u] = i < n ? from[i] : 0;
        }
        last = lanes_join<64>(last, Smaller{});
        __syncthreads();
        if ((threadIdx.x & 63) == 0) low[threadIdx.x >> 6] = last;
        if (threadIdx.x == 0) number = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) last = min(last, low[w]);
#pragma unroll
        for (int u = 0; u < EACH; u++)
            if (held[u] != 0 && (unsigned)(held[u] >> 32) >= last) entries[atomicAdd(&number, 1)] = held[u];
        __syncthreads();
        const TopOut<T> to = {x + row * V, out != nullptr ? nullptr : values + row * k, out != nullptr ? nullptr : places + row * k,
                              out != nullptr ? out + job * k : nullptr};
        const int here = min(number, k);  // (fewer than k: the row's last part, short and alone in its group)
        top_order_out<512>(entries, number, here, to);
        if (out != nullptr)
            for (int i = here + (int)threadIdx.x; i < k; i += 512) out[job * k + i] = 0;
    }
}

struct TopPlan {
    long rows, V;
    int k, dtype;
    bool ok() const {
        return rows >= 1 && rows <= 1L << 30 && V >= 1 && V <= 1L << 24 && k >= 1 && k <= kTopMost && k <= V && rows <= (1L << 40) / V && known(dtype);
    }
    // lanes of a row, or 0
    int lanes() const { return V <= 256 && k <= 16 ? 16 : V <= 512 && k <= 32 ? 32 : V <= 1024 && k <= 64 ? 64 : 0; }
    // Workgroups of 128 threads, more of which a CU has, of no more values than are theirs to sort while others wait (bf16, us, and by 512 threads: 8192 rows of
    // 4000 values, k = 200 88, 161, k = 300 115, 203; 2000 x 1500, k = 200 30, 48, but 16 rows 21.8, 16.8; 2000 x 4000, k = 400 74, 61; 8192 x 8000, k = 400
    // 243, 217)
    bool small() const { return V <= 8192 && (k <= 128 || (k <= 256 && rows > 512) || (k <= 512 && V <= 4096 && rows > 4096)); }
    // parts of a row: where rows are few, no fewer than 4096 and 8 k values each
    int parts() const {
        if (lanes() != 0 || V <= 8192) return 1;
        const long least = std::max(4096L, 8L * k), most = V / least, want = (512 + rows - 1) / rows;
        return (int)std::max(std::min(most, want), 1L);
    }
    long length() const { return ((V + parts() - 1) / parts() + 7) / 8 * 8; }
};
static unsigned top_blocks(long n) { return (unsigned)std::min(n, 1L << 20); }
template <typename T>
static int top_typed(const TopPlan &p, const T *x, T *values, long long *places, Arena &ws, hipStream_t st) {
    if (const int lanes = p.lanes(); lanes != 0) {
        if (ws.dry()) return 0;
        const long each = (p.V + lanes - 1) / lanes;
        auto *kernel = lanes == 16   ? each <= 4    ? top_lanes_kernel<T, 16, 4>
                                       : each <= 8  ? top_lanes_kernel<T, 16, 8>
                                       : each <= 12 ? top_lanes_kernel<T, 16, 12>
                                                    : top_lanes_kernel<T, 16, 16>
                       : lanes == 32 ? each <= 8 ? top_lanes_kernel<T, 32, 8> : top_lanes_kernel<T, 32, 16>
                                     : each <= 8 ? top_lanes_kernel<T, 64, 8> : top_lanes_kernel<T, 64, 16>;
        const long per = 256 / lanes;
        kernel<<<dim3(top_blocks((p.rows + per - 1) / per)), dim3(256), 0, st>>>(x, values, places, p.rows, (int)p.V, p.k);
        return status();
    }
    const long length = p.length();
    int parts = (int)((p.V + length - 1) / length);
    const size_t room = (size_t)p.rows * parts * p.k * sizeof(u64);
    u64 *in = parts > 1 ? (u64 *)ws.take(room) : nullptr, *out = parts > 1 ? (u64 *)ws.take(room) : nullptr;
    if (ws.dry()) return 0;
    if (p.small())
        top_kernel<T, 128><<<dim3(top_blocks(p.rows)), dim3(128), 0, st>>>(x, values, places, in, p.rows, p.V, p.k, 1, length);
    else
        top_kernel<T, 512><<<dim3(top_blocks(p.rows * parts)), dim3(512), 0, st>>>(x, values, places, in, p.rows, p.V, p.k, parts, length);
    int e = status();
    while (parts > 1 && e == 0) {
        const int group = kJoinEntries / p.k, after = (parts + group - 1) / group;
        top_join_kernel<T><<<dim3(top_blocks(p.rows * after)), dim3(512), 0, st>>>(in, x, values, places, after > 1 ? out : nullptr, p.rows, p.V, p.k,
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
