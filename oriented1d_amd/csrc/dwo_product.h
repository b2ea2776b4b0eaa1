// Matrix products of the operators around wide layers: the gated feed-forward block (dwo_gated.hip), the cross entropy of many classes
// (dwo_head.hip) and layers with 8-bit checkpoints (dwo_check8.hip).
//
//   D[m][n] = sum_k A[m][k] * B[n][k]   with an epilogue on the sums while they are in registers.
//
// Either operand lies in memory with k fast (A [M][K]) or with k slow (A [K][M], what the product of a gradient reads), so that no
// tensor is transposed.  Values are 16 bits wide, sums 32.  fp32 operands come as three planes of bf16 whose sum they are (8 + 8 + 8
// bits of mantissa, planes_of), and their product is six of the nine products of planes, small ones first: what is left out, two products of
// 2^-8 and 2^-17 at the most of their operands, is 2^-24 of a product at the most and of either sign.  417 TFLOP/s at best, where the fp32
// matrix instructions give 157, at the accuracy of sums in fp32.
#pragma once

#include <utility>

#include "dwo_linear.h"

namespace dwo {

struct Operand {  // rows of `pitch` values (a multiple of eight), 16-byte aligned; `plane` values from one plane to the next
    const void *p;
    long pitch, plane;
    int planes;  // 1, 2 (halves of 16-bit operands made between products) or 3 (fp32)
};
struct Product {
    Operand a, b;
    long M, N, K;
    long gap;  // gated weights: values from the row of a gate to that of what it multiplies (0: rows as they come)
    int pairs;
    unsigned codes_a, codes_b;  // the planes of each pair, two bits a pair
    unsigned summed;            // the pairs, a bit each, whose planes of A are in its sums
    int mtiles, ntiles, splits;
    int per, steps;  // steps of 64 per split, in all
};

// (2,0) (0,2) (1,1) (1,0) (0,1) (0,0); where one operand has a single plane, the other's planes (two halves meet single planes only)
inline void product_pairs(Product &p) {
    const int a = p.a.planes, b = p.b.planes;
    p.pairs = a == 3 && b == 3 ? 6 : a > b ? a : b;
    p.codes_a = a == 3 && b == 3 ? 0x052 : a == 3 ? 0x006 : a == 2 ? 0x001 : 0;
    p.codes_b = a == 3 && b == 3 ? 0x118 : b == 3 ? 0x006 : b == 2 ? 0x001 : 0;
    p.summed = a == 3 && b == 3 ? 0x29 : b == 3 ? 0x4 : 0x7;
}

// ------------------------------------------------------------------------------------------------- stages in LDS
constexpr int kProdK = 64;  // summed indices of a stage

// R rows (k fast) or columns (k slow) of an operand, 64 summed indices, straight to LDS: sixteen bytes per lane and load, zeros beyond
// the operand's ends.  k fast: rows of 128 bytes whose 16-byte pieces are permuted by the row (lin_fragment).  k slow: 64 rows of R
// values whose 32-byte units are permuted by the row, so that the eight rows of a transposing read lie on different banks.
// HALF > 0: rows come in runs of HALF gates and the HALF rows that these multiply.
__device__ __forceinline__ int prod_key(int row, int R) {
    return R >= 128 ? (row & 3) | (row >> 1 & 4) : R == 64 ? (row >> 1 & 1) | (row >> 2 & 2) : row >> 3 & 1;
}
template <int R, int THREADS, bool SLOW, int HALF>
struct Stage {
    static constexpr int U = R * 8 / THREADS, ROWS = THREADS / (R / 8);
    // k slow: a lane's rows are ROWS apart, and their permutation is the same every sixteen rows
    static constexpr int OFFS = SLOW ? (ROWS % 16 == 0 ? 1 : 16 / ROWS) : U;
    static_assert(R * 8 % THREADS == 0 && THREADS % 64 == 0 && (!SLOW || U % OFFS == 0), "whole loads");
    const char *base, *at;  // of plane 0, and where the next stage comes from (k slow) or its plane (k fast)
    long plane, gap, step;  // bytes
    unsigned off[OFFS], pitch;
    // (a row or column that the operand has not is nowhere: every other access lies inside it)
    __device__ __forceinline__ void init(const Operand &o, long rows, long r0, long skip) {
        plane = o.plane * 2, gap = skip * 2, step = kProdK * o.pitch * 2, pitch = (unsigned)o.pitch * 2;
        if constexpr (SLOW) {
            base = reinterpret_cast<const char *>(o.p) + r0 * 2;
#pragma unroll
            for (int u = 0; u < OFFS; u++) {
                const int q = threadIdx.x % (R / 8), c = ((q >> 1) ^ prod_key(row(u), R)) * 16 + (q & 1) * 8;
                off[u] = r0 + c < o.pitch ? (unsigned)row(u) * pitch + (unsigned)c * 2 : kLinNowhere;
            }
        } else {
            base = reinterpret_cast<const char *>(o.p) + r0 * o.pitch * 2;
#pragma unroll
            for (int u = 0; u < U; u++) off[u] = r0 + row(u) < rows ? (unsigned)row(u) * pitch + piece() * 16 : kLinNowhere;
        }
        at = base;
    }
    static __device__ __forceinline__ int row(int u) {
        const int f = (int)threadIdx.x + u * THREADS, s = SLOW ? f / (R / 8) : f / 8;
        return HALF > 0 ? s / (2 * HALF) * HALF + s % HALF : s;
    }
    static __device__ __forceinline__ int piece() { return (threadIdx.x % 8) ^ (threadIdx.x / 8 % 8); }
    __device__ __forceinline__ void seek(int which, long k0) { at = base + which * plane + (SLOW ? k0 / kProdK * step : 0); }
    // load u of a stage.  left: summed indices from k0 to the operand's end; beyond it a lane reads nowhere, which writes zeros
    __device__ __forceinline__ void load(uint16_t *lds, int k0, int left, int u) const {
        typedef __attribute__((address_space(3))) void lds_void;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#ifdef __HIP_DEVICE_COMPILE__
        const bool second = HALF > 0 && (wave * 8 + u * (THREADS / 8)) / (HALF > 0 ? HALF : 1) % 2 != 0;
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(second ? at + gap : at), 0, 0x7fffffff, 0x00020000);
        const unsigned from = SLOW ? ((int)threadIdx.x / (R / 8) < left - u * ROWS ? off[u % OFFS] : kLinNowhere)
                                   : off[u] | (piece() * 8 < left ? 0u : kLinNowhere);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void *)(lds + (wave * 64 + u * THREADS) * 8), 16, from,
                                                 SLOW ? (int)(u / OFFS * OFFS * ROWS * pitch) : k0 * 2, 0, 0);
#endif
    }
    __device__ __forceinline__ void advance() {
        if constexpr (SLOW) at += step;
    }
};

// A wave's fragments of a stage: sixteen rows (columns) each, from slot0 (a multiple of sixteen times their number, a power of two) on, x
// 32 summed indices, 32 kk .. of the stage; a lane's eight values are 8 g .. of row c.
template <int R, bool SLOW>
struct Fragments {
    unsigned at;  // where the lane reads of fragment 0 (k slow), bytes; the others' places differ in single bits
    int slot;
    __device__ __forceinline__ void init(int slot0) {
        slot = slot0;
        if constexpr (SLOW) {
            const int lane = threadIdx.x & 63, i = lane & 15, row = 8 * (lane >> 4) + (i >> 2);
            at = 2 * ((unsigned)(row * R + prod_key(row, R) * 16 + (i & 3) * 4) ^ (unsigned)slot0);
        }
    }
    // (the places are made anew each time, one instruction each: kept, they cost the registers that the fragments need)
    __device__ __forceinline__ void start() {
        if constexpr (SLOW) asm volatile("" : "+v"(at));
    }
    __device__ __forceinline__ mma_s8 read(const uint16_t *lds, int f, int kk) const {
        if constexpr (SLOW) {
            typedef __attribute__((address_space(3))) mma_s4 lds_s4;
            const char *from = reinterpret_cast<const char *>(lds) + (at ^ (unsigned)(32 * f)) + 64 * kk * R;
            const mma_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)from);
            const mma_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(from + 8 * R));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return lin_fragment<kProdK>(lds, slot + 16 * f, kk);
        }
    }
};

// ------------------------------------------------------------------------------------------------- what goes out
enum { OUT_F32 = 0, OUT_BF16 = 1, OUT_F16 = 2, OUT_PLANES = 3 };  // (the first three are the DWO_ codes)
struct Out {
    void *p;
    long pitch, plane;
    int type;
};
__device__ __forceinline__ uint16_t bits16(int type, float v) {
    return type == OUT_F16 ? __builtin_bit_cast(uint16_t, from_float<f16_t>(v)) : from_float<bf16_t>(v).bits;
}
__device__ __forceinline__ unsigned pack16(int type, float a, float b) {
    return type == OUT_F16 ? lin_pack<f16_t>(a, b) : pack_bf16(a, b);
}
__device__ __forceinline__ float bf16_value(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ float bf16_nearest(float v) { return bf16_value(from_float<bf16_t>(v).bits); }
// v's three planes, each the nearest value of eight bits to what those before it leave (what the products of planes leave out has either sign
// then; with planes cut toward zero it is 0.6 2^-24 of a product in the mean and up to 8, always toward zero).  Infinities and NaN are in
// the last one, which meets nothing but the other operand's first, whose sign and zeros are the operand's own: the products are infinite
// where those of fp32 are.  In front of them is 1 with their sign, so that this holds for two infinities as well.
__device__ __forceinline__ void planes_of(float v, float (&q)[3]) {
    const bool finite = __builtin_fabsf(v) < INFINITY;
    q[0] = bf16_nearest(v);
    // (the largest numbers do not become infinite)
    if (finite && __builtin_fabsf(q[0]) == INFINITY) q[0] = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
    const float r = v - q[0];
    q[1] = bf16_nearest(r);
    q[2] = r - q[1];
    if (!finite) q[0] = __builtin_copysignf(1.f, v), q[1] = 0.f, q[2] = v;
}
__device__ __forceinline__ void out_one(const Out &o, long m, long n, float v) {
    const size_t at = (size_t)m * o.pitch + n;
    if (o.type == OUT_F32) {
        reinterpret_cast<float *>(o.p)[at] = v;
    } else if (o.type == OUT_PLANES) {
        float q[3];
        planes_of(v, q);
#pragma unroll
        for (int e = 0; e < 3; e++) reinterpret_cast<uint16_t *>(o.p)[at + e * o.plane] = from_float<bf16_t>(q[e]).bits;
    } else {
        reinterpret_cast<uint16_t *>(o.p)[at] = bits16(o.type, v);
    }
}
__device__ __forceinline__ bool out_wide(const Out &o) {
    return o.pitch % (o.type == OUT_F32 ? 4 : 8) == 0 && ((uintptr_t)o.p & 15) == 0;
}

// Stores of whole lines (STREAM: eight lanes have 128 bytes of a row of 16-bit values) go past the L2: what they write does not fit it, and
// another launch reads it (4096 x 4096 x 64, all of it writing, 17.5 / 15.9 us; 25088 x 1536 x 384 59.4 / 57.3).  Pieces of lines go
// through it (fp32 in two stores per lane: the gated block's first product, 16384 x 1024 x 8192, 466 us past it, 400 so).
template <bool STREAM>
__device__ __forceinline__ void store_out(void *to, const mma_u4 &v) {
    if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<mma_u4 *>(to));
    else *reinterpret_cast<mma_u4 *>(to) = v;
}
// eight neighbours n .. n + 7 of row m (n a multiple of eight), those below N
template <bool STREAM = true>
__device__ __forceinline__ void out_octet(const Out &o, bool wide, long m, long n, long N, const float (&v)[8]) {
    if (!wide || n + 8 > N) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (n + e < N) out_one(o, m, n + e, v[e]);
        return;
    }
    const size_t at = (size_t)m * o.pitch + n;
    if (o.type == OUT_F32) {
        mma_f4 *to = reinterpret_cast<mma_f4 *>(reinterpret_cast<float *>(o.p) + at);
        to[0] = mma_f4{v[0], v[1], v[2], v[3]}, to[1] = mma_f4{v[4], v[5], v[6], v[7]};
        return;
    }
    uint16_t *to = reinterpret_cast<uint16_t *>(o.p) + at;
    if (o.type == OUT_PLANES) {
        float q[8][3];
#pragma unroll
        for (int e = 0; e < 8; e++) planes_of(v[e], q[e]);
#pragma unroll
        for (int k = 0; k < 3; k++)
            store_out<STREAM>(to + k * o.plane, mma_u4{pack_bf16(q[0][k], q[1][k]), pack_bf16(q[2][k], q[3][k]), pack_bf16(q[4][k], q[5][k]), pack_bf16(q[6][k], q[7][k])});
        return;
    }
    store_out<STREAM>(to, mma_u4{pack16(o.type, v[0], v[1]), pack16(o.type, v[2], v[3]), pack16(o.type, v[4], v[5]), pack16(o.type, v[6], v[7])});
}
// Eight neighbours of an operand's row; in two halves (o.plane of 16-bit values) the second is what the first one's rounding leaves.  It has
// the first one's sign and is not zero, for which the first goes a step down where it has to (the second is then at most 3/2 steps and not
// 1/2, its own rounding twice as far): an infinite value of the other operand, whose products with both halves are added, is infinite in the sum
// and not NaN.  The second half of infinities and NaN is 1 with their sign.
__device__ __forceinline__ void halves_of(int type, float v, float &first, float &second) {
    auto value = [&](uint16_t b) { return type == OUT_F16 ? to_float(__builtin_bit_cast(f16_t, b)) : bf16_value(b); };
    const uint16_t b = bits16(type, v);
    float h = value(b), rest = v - h;
    const float r = value(bits16(type, rest));
    const bool apart = r == 0.f || ((__float_as_uint(r) ^ __float_as_uint(h)) >> 31) != 0;
    const bool finite = __builtin_fabsf(h) < INFINITY;
    if (apart && (b & 0x7fff) > 1) h = value(b - 1), rest = v - h;
    first = finite ? h : v, second = finite ? rest : __builtin_copysignf(1.f, v);
}
template <bool STREAM = true>
__device__ __forceinline__ void operand_octet(const Out &o, long m, long n, long N, const float (&v)[8]) {
    out_octet<STREAM>(o, true, m, n, N, v);
    if (__builtin_expect(o.type == OUT_PLANES || o.plane == 0, 1)) return;
    // (rare, and behind the first store, whose half is written again: with these values in front of it the gated block's product behind dy, 16384 x
    // 4096 from 1024, which has no second halves, takes 12 of 328 us more)
    float first[8], second[8];
#pragma unroll
    for (int e = 0; e < 8; e++) halves_of(o.type, v[e], first[e], second[e]);
    out_octet<STREAM>(o, true, m, n, N, first);
    out_octet<STREAM>({reinterpret_cast<uint16_t *>(o.p) + o.plane, o.pitch, 0, o.type}, true, m, n, N, second);
}
// one value of an operand
__device__ __forceinline__ void operand_one(const Out &o, long m, long n, float v) {
    if (o.type == OUT_PLANES || o.plane == 0) {
        out_one(o, m, n, v);
        return;
    }
    float first, second;
    halves_of(o.type, v, first, second);
    out_one(o, m, n, first);
    out_one({reinterpret_cast<uint16_t *>(o.p) + o.plane, o.pitch, 0, o.type}, m, n, second);
}

// An epilogue E has
//   begin(p, n): what a lane keeps for its eight columns (n: the first) while it goes down the rows
//   kRow, row(p, m, n0, k): numbers of a row that wait in LDS from the start of the kernel (n0: the tile's first column)
//   load(p, m, n): what the epilogue reads for an octet, asked for one octet ahead
//   octet(p, lane, rows, data, split, m, n, v): eight neighbours of a row; all lanes call it for some row, beyond the ends as well
//   kSums, emit_sum: see SumsEpi
// or, where it writes next to nothing, kDirect and emit(p, lane, rows, m, n0, v): a row's fragments as they are in registers, columns
// n0 + 16 i + 4 g + r, with begin(p, n0) of the wave's first column.
struct Nothing {};

struct Values {  // a vector of fp32 or 16-bit values, or none
    const void *p;
    int type;
    __device__ __forceinline__ float at(long i) const {
        if (type == OUT_F32) return reinterpret_cast<const float *>(p)[i];
        const uint16_t b = reinterpret_cast<const uint16_t *>(p)[i];
        return type == OUT_F16 ? to_float(__builtin_bit_cast(f16_t, b)) : bf16_value(b);
    }
};

// exp(v): v_exp_f32 of v log2(e) with what the product's rounding leaves (relative error 1e-7 where a bare product's grows with |v|)
__device__ __forceinline__ float prod_exp(float v) {
    const float t = v * 1.44269504f;
    const float r = __builtin_fmaf(v, 1.44269504f, -t) + v * 1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(t);
    // From 88.72 on (exp overflows at 88.7228) e is infinite and, r being of either sign, e + e r would not be a number; below -88.72 e is no
    // normal number, and r of infinities is none
    return __builtin_fabsf(v) < 88.72f ? __builtin_fmaf(e, r * 0.693147181f, e) : e;
}

// The plain epilogue: out = alpha * sum + bias[n] + before[m][n].  With several splits the sums go to `part` as they are, and
// product_reduce_kernel does the rest.  sums: the sums over k of A alone (a bias gradient), alpha times.
struct PlainEpi {
    static constexpr bool kSums = false, kDirect = false;
    Out out, sums;      // (sums.p null: none)
    Values bias;        // (p null: none)
    const float *before;  // [M][pitch of out], or null
    const float *alpha, *over;  // alpha = factor * alpha[0] / over[0], 0 where over[0] is 0 (null: 1)
    float factor;
    float *part;        // [splits][M][N], then [splits][M]
    long rows_from, rows_skip;  // output rows from rows_from on lie rows_skip further up; those skipped are not written (0: none)
    long tail;          // columns of A that are only padding (behind rows_from - rows_skip .. rows_from)
    __device__ __forceinline__ long place(long m) const {  // of row m, or -1
        if (rows_skip == 0) return m;
        if (m < rows_from - rows_skip) return m;
        if (m < rows_from) return -1;
        return m - rows_skip < tail ? m - rows_skip : -1;
    }
    __device__ __forceinline__ float scale() const {
        const float a = alpha != nullptr ? alpha[0] * factor : factor;
        return over == nullptr ? a : over[0] > 0.f ? a / over[0] : 0.f;
    }
    __device__ __forceinline__ float finish(long m, long n, float v, float a) const {
        v = __builtin_fmaf(v, a, bias.p != nullptr ? bias.at(n) : 0.f);
        if (before != nullptr) v += before[(size_t)m * out.pitch + n];
        return v;
    }
    struct Lane {
        float bias[8], alpha;
        bool wide;
    };
    __device__ __forceinline__ Lane begin(const Product &p, long n) const {
        Lane l;
        l.alpha = part == nullptr ? scale() : 1.f;
        l.wide = part != nullptr ? p.N % 4 == 0 : out_wide(out);
#pragma unroll
        for (int e = 0; e < 8; e++) l.bias[e] = bias.p != nullptr && part == nullptr && n + e < p.N ? bias.at(n + e) : 0.f;
        return l;
    }
    static constexpr int kRow = 0;
    __device__ __forceinline__ Nothing load(const Product &, long, long) const { return {}; }
    __device__ __forceinline__ void octet(const Product &p, const Lane &l, const unsigned *, const Nothing &, int split, long m, long n,
                                          float (&v)[8]) const {
        if (m >= p.M || n >= p.N) return;
        if (part != nullptr) {
            out_octet({part + (size_t)split * p.M * p.N, p.N, 0, OUT_F32}, l.wide, m, n, p.N, v);
            return;
        }
        const long to = place(m);
        if (to < 0) return;
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = __builtin_fmaf(v[e], l.alpha, l.bias[e]);
        if (before != nullptr)
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (n + e < p.N) v[e] += before[(size_t)to * out.pitch + n + e];
        out_octet(out, l.wide, to, n, p.N, v);
    }
    __device__ __forceinline__ void emit_sum(const Product &p, int split, long m, float v) const {
        if (m >= p.M) return;
        if (part != nullptr) {
            part[(size_t)p.splits * p.M * p.N + (size_t)split * p.M + m] = v;
            return;
        }
        const long to = place(m);
        if (to >= 0) out_one(sums, 0, to, v * scale());
    }
};

struct SumsEpi : PlainEpi {
    static constexpr bool kSums = true;
};

// ------------------------------------------------------------------------------------------------- the product
// Tiles of BM x BN, WM x WN waves.  A stage is 64 summed indices of both operands, two stages in LDS.  While a wave multiplies one
// part of a stage it reads the fragments of the next: a stage is four parts (or eight), half of the wave's rows x half of the stage each.  The one
// barrier of a step comes before the last part, when every wave has the rest of its stage in registers: the stage's LDS takes the
// stage after the next, and the products of that part cover the reads of the next stage's first.
template <int BM_, int BN_, int WM_, int WN_, int WAVES, int STAGES_>
struct Shape {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, THREADS = 64 * WM_ * WN_, PER_SIMD = WAVES, STAGES = STAGES_;
    static constexpr int MF = BM_ / WM_ / 16, NF = BN_ / WN_ / 16;
};
typedef Shape<256, 256, 2, 4, 2, 2> LargeTile;   // 128 KB of LDS, one workgroup per CU
typedef Shape<128, 128, 2, 2, 2, 2> MediumTile;  // 64 KB, two
// The same where no CU has two: twice the waves, and four stages (2048 x 2048 x 2048: 21 us, as the former 27; both transposed 23, 30)
typedef Shape<128, 128, 4, 2, 2, 4> AloneTile;   // 128 KB
// The same for short sums, whose first loads and last stores are much of a tile's time: twice the waves (25088 x 1536 x 384: 45 us, as
// MediumTile 48; x 64 34.5, 39.4; 4096 x 4096 x 768 29.1, 30.4; x 2048
// 63, 61; two gradients of 32768 rows, 256 columns and 150 classes 21.4, 24.3).  Not where an epilogue reads, which half the registers delay (the gated
// block's product behind dy, 3136 x 2048 from 768, 39.5, 37.4)
typedef Shape<128, 128, 4, 2, 4, 2> ShortTile;
constexpr long kShortSteps = 16;
// Few tiles leave most of a CU's LDS free and their waves waiting for memory: more stages on their way
typedef Shape<64, 64, 2, 2, 2, 4> SmallTile;     // 64 KB
typedef Shape<32, 32, 2, 2, 2, 8> ThinTile;      // 64 KB

// f(0), f(1), .. with constant indices, one after the other
template <class F, int... I>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F &&f) {
    ((f(std::integral_constant<int, I>{}), __builtin_amdgcn_sched_barrier(0)), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F &&f) {
    each_of(std::make_integer_sequence<int, N>{}, f);
}
// f(0), f(1), .. until one is false
template <class F, int... I>
__device__ __forceinline__ bool stages_of(std::integer_sequence<int, I...>, F &&f) {
    return (f(std::integral_constant<int, I>{}) && ...);
}

// The LDS of a workgroup: arrays of their own, so that a read of one waits for no load into another
#define DWO_STAGES(S)                                                                                  \
    constexpr int kStageSize = (S::BM + S::BN) * kProdK;                                               \
    __shared__ __attribute__((aligned(16))) uint16_t s0[kStageSize];                                   \
    __shared__ __attribute__((aligned(16))) uint16_t s1[kStageSize];                                   \
    __shared__ __attribute__((aligned(16))) uint16_t s2[S::STAGES > 2 ? kStageSize : 8];               \
    __shared__ __attribute__((aligned(16))) uint16_t s3[S::STAGES > 2 ? kStageSize : 8];               \
    __shared__ __attribute__((aligned(16))) uint16_t s4[S::STAGES > 4 ? kStageSize : 8];               \
    __shared__ __attribute__((aligned(16))) uint16_t s5[S::STAGES > 4 ? kStageSize : 8];               \
    __shared__ __attribute__((aligned(16))) uint16_t s6[S::STAGES > 4 ? kStageSize : 8];               \
    __shared__ __attribute__((aligned(16))) uint16_t s7[S::STAGES > 4 ? kStageSize : 8];               \
    const Stages lds = {s0, s1, s2, s3, s4, s5, s6, s7}
struct Stages {
    uint16_t *s0, *s1, *s2, *s3, *s4, *s5, *s6, *s7;
};

// Workgroup `block` of `blocks` (a multiple of eight).  lrow: room for the rows' numbers.
template <typename T, class S, bool AS, bool BS, bool GATED, class Epi>
__device__ __forceinline__ void product_body(const Product &p, const Epi &epi, int block, int blocks, const Stages &lds, unsigned *lrow) {
    constexpr int BM = S::BM, BN = S::BN, MF = S::MF, NF = S::NF, SF = MF / S::WN > 0 ? MF / S::WN : 1;
    constexpr bool SUMS = Epi::kSums;
    constexpr int STAGES = S::STAGES, SIZE = (BM + BN) * kProdK;
    auto stage = [&](auto i) -> uint16_t * {
        constexpr int k = decltype(i)::value % STAGES;
        if constexpr (k == 0) return lds.s0;
        else if constexpr (k == 1) return lds.s1;
        else if constexpr (k == 2) return lds.s2;
        else if constexpr (k == 3) return lds.s3;
        else if constexpr (k == 4) return lds.s4;
        else if constexpr (k == 5) return lds.s5;
        else if constexpr (k == 6) return lds.s6;
        else return lds.s7;
    };
    // an XCD (workgroup ids modulo eight) takes a run of tiles; runs go down groups of rows of tiles, so that the tiles of an XCD
    // at one time share both operands' lines
    const int per = blocks / 8, id = block % 8 * per + block / 8;
    const int tiles = p.mtiles * p.ntiles;
    const int split = id / tiles, tile = id % tiles;
    if (split >= p.splits) return;
    constexpr int GROUP = 8;
    const int group = tile / (GROUP * p.ntiles), in = tile % (GROUP * p.ntiles), high = min(GROUP, p.mtiles - group * GROUP);
    const int mt = group * GROUP + in % high, nt = in / high;
    const long m0 = (long)mt * BM, n0 = (long)nt * BN;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;
    Stage<BM, S::THREADS, AS, 0> sa;
    Stage<BN, S::THREADS, BS, GATED ? 8 * NF : 0> sb;
    sa.init(p.a, p.M, m0, 0);
    sb.init(p.b, GATED ? p.N / 2 : p.N, GATED ? n0 / 2 : n0, p.gap);
    mma_f4 acc[NF][MF], accs[SF];
#pragma unroll
    for (int i = 0; i < NF; i++)
#pragma unroll
        for (int j = 0; j < MF; j++) acc[i][j] = mma_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < SF; j++) accs[j] = mma_f4{0.f, 0.f, 0.f, 0.f};

    if constexpr (Epi::kRow > 0)
        if ((int)threadIdx.x < BM && m0 + (int)threadIdx.x < p.M)
#pragma unroll
            for (int k = 0; k < Epi::kRow; k++) lrow[threadIdx.x * Epi::kRow + k] = epi.row(p, m0 + (int)threadIdx.x, n0, k);
    const int ksteps = (int)((p.K + kProdK - 1) / kProdK);
    const int first = split * p.per, count = min(p.per, p.steps - first);
    int pair = first / ksteps, k0 = first % ksteps * kProdK, more = count;
    sa.seek(p.codes_a >> (2 * pair) & 3, k0), sb.seek(p.codes_b >> (2 * pair) & 3, k0);
    // the loads of the next stage, U in all; (a loop of one body: an odd last step is followed by one of zeros)
    constexpr int UA = decltype(sa)::U, U = UA + decltype(sb)::U;
    auto load = [&](uint16_t *to, int u) {
        const int left = more > 0 ? (int)p.K - k0 : 0;
        if (u < UA) sa.load(to, k0, left, u);
        else sb.load(to + BM * kProdK, k0, left, u - UA);
    };
    auto loaded = [&] {
        sa.advance(), sb.advance();
        k0 += kProdK, more--;
        if (k0 >= p.K) {
            k0 = 0, pair++;
            sa.seek(p.codes_a >> (2 * pair) & 3, 0), sb.seek(p.codes_b >> (2 * pair) & 3, 0);
        }
    };
    auto fetch = [&](uint16_t *to) {
#pragma unroll
        for (int u = 0; u < U; u++) load(to, u);
        loaded();
    };
    // (quarters of eight fragments and not halves: sixteen registers less, which two transposing operands have not)
    constexpr int Q = MF == 8 ? 4 : MF > 1 ? 2 : 1, MH = MF / Q;
    mma_s8 fa[4][MH], fb[2][NF];  // (at most three of the four hold anything at one time)
    Fragments<BM, AS> part_a;
    Fragments<BN, BS> part_b;
    part_a.init(wm * MF * 16), part_b.init(wn * NF * 16);
    // part t of a stage: q of Q of the rows and half kk; its A goes to fa[t % 4], its B to fb[kk] (with the first rows)
    constexpr int G = MH * NF;  // products of a part
    static_assert(Q > 1 || G == 1);  // (a part alone in its half reads over itself: behind its only product)
    auto multiply = [&](int t, int k) {
        const int kk = t / Q, q = t % Q, j = k / NF, i = k % NF;
        acc[i][q * MH + j] = Mma<T>::run(fb[kk][i], fa[t % 4][j], acc[i][q * MH + j]);
    };
    auto reads = [&](int t) { return t % Q == 0 ? MH + NF : MH; };
    auto read = [&](const uint16_t *from, int t, int r) {
        const int kk = t / Q, q = t % Q;
        if (r < MH) {
            if (r == 0) part_a.start();
            fa[t % 4][r] = part_a.read(from, q * MH + r, kk);
        } else {
            if (r == MH) part_b.start();
            fb[kk][r - MH] = part_b.read(from + BM * kProdK, r - MH, kk);
        }
    };
    auto read_all = [&](const uint16_t *from, int t) {
#pragma unroll
        for (int r = 0; r < MH + NF; r++)
            if (r < reads(t)) read(from, t, r);
    };
    // sums over A alone, in the workgroups of the first column of tiles: products with ones, with zeros elsewhere and where a plane of A
    // meets another than B's first, once more (a branch would cost more than these products, one in sixteen of all).  Where A's only plane
    // meets both halves of B, with 1/2 both times: its infinities are not to meet zeros (of three planes the one that holds them does not)
    int at_pair = first / ksteps, at_step = first % ksteps;
    Fragments<BM, AS> sums_of;
    sums_of.init((wm * MF + wn * SF % MF) * 16);
    const short unit = nt != 0 ? 0 : p.b.planes == 2 ? Mma<T>::kHalf : Mma<T>::kOne;
    auto add_sums = [&](const uint16_t *la) {
        if constexpr (SUMS) {
            const short one = p.summed >> at_pair & 1 ? unit : 0;
            at_step++;
            const bool wrap = at_step == ksteps;
            at_step = wrap ? 0 : at_step, at_pair = wrap ? at_pair + 1 : at_pair;
            const mma_s8 ones = {one, one, one, one, one, one, one, one};
            sums_of.start();
#pragma unroll
            for (int kk = 0; kk < 2; kk++)
#pragma unroll
                for (int j = 0; j < SF; j++)
                    accs[j] = Mma<T>::run(ones, sums_of.read(la, j, kk), accs[j]);
        }
    };
    // all but the last `stages` stages' loads of this wave have arrived, and what it read of LDS
    auto wait = [](auto stages) {
        constexpr int n = decltype(stages)::value * (decltype(sa)::U + decltype(sb)::U);
        static_assert(n < 64, "what the counter holds");
        __builtin_amdgcn_s_waitcnt(0x0070 | (n & 15) | n >> 4 << 14);
        asm volatile("s_barrier" ::: "memory");
    };
    // What goes out between the products of a part, evenly: the reads of the part after the next, in the last two the loads too (8192 x 8192 x
    // 8192 in bf16: 859 us, with the reads of the next part only 872; transposing operands 964, and 987)
    auto step = [&](auto i) {
        uint16_t *current = stage(i);
        const uint16_t *next = stage(std::integral_constant<int, decltype(i)::value + 1>{});
        add_sums(current);
#pragma unroll
        for (int t = 0; t < 2 * Q; t++) {
            // this wave's reads of the stage are done, and its part of the next one is there; so are the other waves' behind the barrier
            if (t == 2 * Q - 2) wait(std::integral_constant<int, STAGES - 2>{});
            const bool late = t >= 2 * Q - 2;
            const int after = late ? t + 2 - 2 * Q : t + 2, n = reads(after), first = (t - (2 * Q - 2)) * G;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int k = 0; k < G; k++) {
                multiply(t, k);
#pragma unroll
                for (int r = 0; r < MH + NF; r++)
                    if (r >= k * n / G && r < (k + 1) * n / G) read(late ? next : current, after, r);
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (late && u >= (first + k) * U / (2 * G) && u < (first + k + 1) * U / (2 * G)) load(current, u);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
        }
        loaded();
    };
    if constexpr (STAGES == 2) {
        fetch(lds.s0);
        wait(std::integral_constant<int, 0>{});
        fetch(lds.s1);
        read_all(lds.s0, 0), read_all(lds.s0, 1);
        for (int s = 0; s < count; s += 2) step(std::integral_constant<int, 0>{}), step(std::integral_constant<int, 1>{});
    } else {
        stages_of(std::make_integer_sequence<int, STAGES>{}, [&](auto i) { return fetch(stage(i)), true; });
        wait(std::integral_constant<int, STAGES - 1>{});
        read_all(lds.s0, 0), read_all(lds.s0, 1);
        int s = 0;
        while (stages_of(std::make_integer_sequence<int, STAGES>{}, [&](auto i) { return step(i), ++s < count; })) {}
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // (nothing may arrive behind the sums)
    if constexpr (Epi::kDirect) {
        // (1141 us through LDS, 1001 so: statistics of 8192 x 1024 x 65536.  Where rows are written their pieces are too short, 64 bytes)
        const long nw = n0 + wn * 16 * NF, mw = m0 + wm * 16 * MF + (threadIdx.x & 15);
        const auto local = epi.template begin<NF>(p, nw);
        each<MF>([&](auto j) {
            mma_f4 v[NF];
#pragma unroll
            for (int i = 0; i < NF; i++) v[i] = acc[i][j];
            epi.emit(p, local, lrow + (wm * 16 * MF + 16 * j + (threadIdx.x & 15)) * Epi::kRow, mw + 16 * j, nw, v);
        });
    } else {
        // The sums go through LDS, each wave's through its own part, and come back as eight neighbours of a row per lane (gated: eight
        // gates and what they multiply): wide stores, row sums over few lanes, and a loop of one body.  Quads of a row are permuted by the row.
        __syncthreads();
        constexpr int QUADS = 4 * NF, PF = MF < 4 ? MF : 4, ROWS = 16 * PF, LANES = GATED ? NF : 2 * NF, STEP = 64 / LANES;
        constexpr int WAVES = S::THREADS / 64, PART = ROWS * 16 * NF, FIT = SIZE / 2 / PART < WAVES ? SIZE / 2 / PART : WAVES;
        static_assert(2 * FIT >= WAVES, "the waves' parts fit two stages");
        float *mine = reinterpret_cast<float *>(wave < FIT ? lds.s0 : lds.s1) + wave % FIT * PART;
        const int lane = threadIdx.x & 63;
        const int o = lane % LANES, row0 = lane / LANES;
        const long nl = (GATED ? n0 / 2 + wn * 8 * NF : n0 + wn * 16 * NF) + o * 8;
        const auto local = epi.begin(p, nl);
        // What the epilogue reads comes two turns ahead (gated block of 16384 x 1024 x 4096 backward: 335 us, one turn ahead 351)
        auto data = epi.load(p, m0 + wm * 16 * MF + row0, nl), next = epi.load(p, m0 + wm * 16 * MF + row0 + STEP, nl);
#pragma unroll
        for (int pass = 0; pass < MF / PF; pass++) {
#pragma unroll
            for (int j = 0; j < PF; j++)
#pragma unroll
                for (int i = 0; i < NF; i++) {
                    const int row = 16 * j + (lane & 15), quad = 4 * i + (lane >> 4);
                    reinterpret_cast<mma_f4 *>(mine)[row * QUADS + (quad ^ (row & (QUADS - 1)))] = acc[i][pass * PF + j];
                }
            auto octet = [&](int row, int at, float (&v)[8]) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const mma_f4 q = reinterpret_cast<const mma_f4 *>(mine)[row * QUADS + ((2 * at + h) ^ (row & (QUADS - 1)))];
#pragma unroll
                    for (int e = 0; e < 4; e++) v[4 * h + e] = q[e];
                }
            };
            const long mp = m0 + wm * 16 * MF + pass * ROWS;
#pragma unroll 2
            for (int row = row0; row < ROWS; row += STEP) {
                const auto now = data;
                data = next;
                if (pass + 1 < MF / PF || row + 2 * STEP < ROWS) next = epi.load(p, mp + row + 2 * STEP, nl);
                const unsigned *rows = lrow + (wm * 16 * MF + pass * ROWS + row) * Epi::kRow;
                float v[8];
                octet(row, o, v);
                if constexpr (GATED) {
                    float u[8];
                    octet(row, NF + o, u);
                    epi.octet(p, local, mp + row, nl, v, u);
                } else {
                    epi.octet(p, local, rows, now, split, mp + row, nl, v);
                }
            }
        }
    }
    if constexpr (SUMS)
        if (nt == 0 && wn * SF < MF && (threadIdx.x & 63) < 16) {
#pragma unroll
            for (int j = 0; j < SF; j++) epi.emit_sum(p, split, m0 + (wm * MF + wn * SF + j) * 16 + (threadIdx.x & 15), accs[j][0]);
        }
}

template <typename T, class S, bool AS, bool BS, bool GATED, class Epi>
__global__ __launch_bounds__(S::THREADS, S::PER_SIMD) void product_kernel(Product p, Epi epi) {
    DWO_STAGES(S);
    __shared__ unsigned lrow[Epi::kRow > 0 ? S::BM * Epi::kRow : 1];
    product_body<T, S, AS, BS, GATED>(p, epi, (int)blockIdx.x, (int)gridDim.x, lds, lrow);
}

// ------------------------------------------------------------------------------------------------- on the host
// A workspace handed out piece by piece.  With no memory behind it, it measures: the calls below then launch nothing.
struct Arena {
    char *base;
    size_t used, size;
    static Arena measure() { return {nullptr, 0, (size_t)-1}; }
    bool dry() const { return base == nullptr; }
    static size_t whole(size_t bytes) { return (bytes + 255) / 256 * 256; }
    bool fits(size_t bytes) const { return whole(bytes) <= size - used; }
    void *take(size_t bytes) {
        void *p = base != nullptr ? base + used : nullptr;
        used += whole(bytes);
        return p;
    }
};
inline long up8(long n) { return (n + 7) / 8 * 8; }
inline int status() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : (int)e;
}
inline unsigned blocks_for(long work, long most = 4096) {
    const long n = (work + 255) / 256;
    return (unsigned)(n < 1 ? 1 : n < most ? n : most);
}
inline size_t size_of(int dtype) { return dtype == DWO_F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == DWO_F32 || dtype == DWO_BF16 || dtype == DWO_F16; }

// Where an operator's forward pass has no more multiply-adds than this, the 16-bit operands that one of its products makes for another are held
// in two halves, 16 bits more, and their rounding is in no result.  Where results are large it takes them from one rounding off to 1.41; of a few
// values by up to twice, and there the second half costs little: forward and backward, bf16, in a graph, gated block 49 x 768 -> 2048 42 us, so 48,
// 784 x 192 -> 512 32, 44, loss of 256 x 768 x 1000 29, 35 (from Python's calls, 75 to 100 us either way); at twice the limit 1000 x 256 -> 680 41, 57,
// 32768 x 96 x 150 56, 74.
constexpr double kHalvesWork = 1 << 28;
// room for an operand of rows x pitch that a kernel writes
inline Operand take_operand(Arena &ws, long rows, long pitch, int dtype, double work = 2 * kHalvesWork) {
    Operand o;
    o.planes = dtype == DWO_F32 ? 3 : work <= kHalvesWork ? 2 : 1;
    o.pitch = pitch, o.plane = rows * pitch;
    o.p = ws.take((size_t)o.planes * o.plane * 2);
    return o;
}
inline Out out_of(const Operand &o, int dtype) {
    return {const_cast<void *>(o.p), o.pitch, o.planes > 1 ? o.plane : 0, dtype == DWO_F32 ? OUT_PLANES : dtype};
}
// Operands that are made before the products of a call, by one launch (dwo_product.hip).
struct StageJob {
    const void *src;
    const uint8_t *exps;  // of a checkpoint (dwo_check8.h), or null
    uint16_t *dst;
    long rows, gate, move, all, pitch, plane;
    int cols, type;
};
struct Staging {
    StageJob jobs[4];
    int count = 0;
    // a dense [rows][cols] matrix as an operand: itself, or a copy that is one.  move > 0: the rows from `gate` on go `move` rows further
    // down (the second half of gated weights whose hidden size is no multiple of eight), with zeros between and behind.
    Operand matrix(const void *src, long rows, long cols, int dtype, Arena &ws, long gate = 0, long move = 0) {
        if (dtype != DWO_F32 && cols % 8 == 0 && move == 0) return {src, cols, 0, 1};
        const Operand o = take_operand(ws, rows + 2 * move, up8(cols), dtype);
        add(o, src, nullptr, rows, cols, move == 0 ? rows : gate, move, dtype);
        return o;
    }
    // the values that a checkpoint holds: one plane whatever the type, they are exact in 16 bits
    Operand held8(const int8_t *codes, const uint8_t *exps, long rows, long cols, int dtype, Arena &ws) {
        const Operand o = take_operand(ws, rows, up8(cols), DWO_BF16);
        add(o, codes, exps, rows, cols, rows, 0, dtype);
        return o;
    }
    int launch(bool dry, hipStream_t st);

private:
    void add(const Operand &o, const void *src, const uint8_t *exps, long rows, long cols, long gate, long move, int type) {
        jobs[count++] = {src, exps, (uint16_t *)const_cast<void *>(o.p), rows, gate, move, rows + 2 * move, o.pitch, o.plane, (int)cols, type};
    }
};

// A [M][K] times B [N][K] with the plain epilogue, whose `part` is filled in here (dwo_product.hip)
int plain_product(const Operand &a, const Operand &b, long M, long N, long K, int dtype, PlainEpi epi, Arena &ws, hipStream_t st);

// Products of a backward pass that do not wait for each other, as one launch: of gradients with weights, A [M][K] times B [K][N], and of
// gradients with activations, A [K][M] times B [K][N].  Their tiles fill the chip together, where each alone leaves a part of its last round.
struct GroupPart {
    Product p;
    PlainEpi epi;
    int kind, blocks;  // 0: A [M][K], 1: A [K][M], 2: that with sums over A
};
struct ProductGroup {
    GroupPart part[3];
    int count = 0;
    void add(bool a_slow, const Operand &a, const Operand &b, long M, long N, long K, const PlainEpi &epi);
    int launch(int dtype, Arena &ws, hipStream_t st);
};

inline PlainEpi plain_epilogue(const Out &out) { return {out, {nullptr, 0, 0, 0}, {nullptr, 0}, nullptr, nullptr, nullptr, 1.f, nullptr, 0, 0, 0}; }

// Workgroups of a launch: it has fewer than 2^32 threads, and these have 512 at most.  Products of more tiles than that take larger ones; of 256 x 256
// it is as many as 2^39 results need.
constexpr long kMostGroups = (1L << 23) - 8;

// products whose epilogue is not the plain one
template <typename T, class S, bool AS, bool BS, bool GATED, class Epi>
int launch_shape(Product p, const Epi &epi, hipStream_t st) {
    p.mtiles = (int)((p.M + S::BM - 1) / S::BM), p.ntiles = (int)((p.N + S::BN - 1) / S::BN);
    const long total = (long)p.mtiles * p.ntiles * p.splits;
    if (total > kMostGroups) return DWO_ERR_BAD_SHAPE;
    product_kernel<T, S, AS, BS, GATED, Epi><<<dim3((unsigned)((total + 7) / 8 * 8)), dim3(S::THREADS), 0, st>>>(p, epi);
    return status();
}
inline long tiles_of(long M, long N, int bm, int bn) { return ((M + bm - 1) / bm) * ((N + bn - 1) / bn); }
inline Product make_product(const Operand &a, const Operand &b, long M, long N, long K, long gap) {
    Product p{a, b, M, N, K, gap, 1, 0, 0, 0, 0, 0, 1, 0, 0};
    product_pairs(p);
    p.steps = p.per = (int)((K + kProdK - 1) / kProdK * p.pairs);
    return p;
}
// Time of a product with square tiles of this size, us: workgroups that have a CU to themselves wait for memory step by step, others
// share its units.  The numbers are fits to 450 bf16 products of 64 to 25088 rows x 384 to 8192 columns x 64 to 16384 summed indices, operands
// of every order, which they meet within 10 % (root of the mean square; 13 % the smallest tile); the tile that they choose is 0.2 % slower
// than the fastest of the four in the geometric mean, 9 % at the most (with MediumTile in AloneTile's place).  First round: a launch with its first loads and last stores, and a
// step; then each round.
struct TileCost {
    int size;
    float first, first_step, more, more_step;
};
constexpr TileCost kTileCosts[4] = {
    {256, 11.6f, 1.19f, 10.f, 1.41f}, {128, 5.8f, 0.49f, 2.65f, 0.44f}, {64, 4.2f, 0.275f, 1.25f, 0.195f}, {32, 4.f, 0.15f, 1.2f, 0.105f}};
inline float tile_time(const TileCost &c, long workgroups, long steps) {
    if (workgroups <= kLinCus) return c.first + (float)steps * c.first_step;
    return 3.5f + (float)((workgroups + kLinCus - 1) / kLinCus) * (c.more + (float)steps * c.more_step);
}
// the tile of a product that is not split
inline int tile_for(long M, long N, long steps) {
    int best = 0;
    for (int i = 1; i < 4; i++) {
        const long tiles = tiles_of(M, N, kTileCosts[i].size, kTileCosts[i].size);
        if (tiles <= kMostGroups && tile_time(kTileCosts[i], tiles, steps) <
                                        tile_time(kTileCosts[best], tiles_of(M, N, kTileCosts[best].size, kTileCosts[best].size), steps))
            best = i;
    }
    return kTileCosts[best].size;
}
template <class E>
constexpr bool epilogue_reads() {
    if constexpr (E::kDirect) return false;
    else return !std::is_same<decltype(std::declval<E>().load(std::declval<Product>(), 0, 0)), Nothing>::value;
}
// f(shape) for tiles of this size in so many workgroups of so many steps, with epilogue E
template <class E, class F>
inline int with_tile(int tile, long workgroups, long steps, F &&f) {
    switch (tile) {
        case 256: return f(LargeTile{});
        case 128:
            if (workgroups <= kLinCus) return f(AloneTile{});
            if constexpr (!epilogue_reads<E>())
                if (steps <= kShortSteps) return f(ShortTile{});
            return f(MediumTile{});
        case 64: return f(SmallTile{});
        default: return f(ThinTile{});
    }
}
// columns of a wave
inline int wave_columns(int tile) { return tile == 32 ? 16 * ThinTile::NF : tile == 64 ? 16 * SmallTile::NF : 16 * LargeTile::NF; }
template <typename T, bool AS, bool BS, bool GATED, class Epi>
int launch_tiles(const Product &p, const Epi &epi, hipStream_t st) {
    const int tile = tile_for(p.M, p.N, p.steps);
    return with_tile<Epi>(tile, tiles_of(p.M, p.N, tile, tile), p.steps,
                     [&](auto shape) { return launch_shape<T, decltype(shape), AS, BS, GATED>(p, epi, st); });
}
template <bool AS, bool BS, bool GATED, class Epi>
int launch_product(const Product &p, int dtype, const Epi &epi, hipStream_t st) {
    if (dtype == DWO_F16) return launch_tiles<f16_t, AS, BS, GATED>(p, epi, st);
    return launch_tiles<bf16_t, AS, BS, GATED>(p, epi, st);
}

}  // namespace dwo
