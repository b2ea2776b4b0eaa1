// Operands of the products around wide layers, and the products with the plain epilogue.
#include <cmath>
#include <utility>

#include "dwo_check8.h"
#include "dwo_product.h"

namespace dwo {

// Eight neighbours per thread: columns padded with zeros to `pitch`, fp32 taken apart into three planes, checkpoints taken out of theirs.
template <typename S>
__device__ __forceinline__ void read_octet(const S *at, int c, int cols, bool real, S (&v)[8]) {
    if (real && cols % (16 / (int)sizeof(S)) == 0 && c + 8 <= cols && sizeof(S) > 1) {
#pragma unroll
        for (int e = 0; e < (int)sizeof(S) / 2; e++) reinterpret_cast<mma_u4 *>(v)[e] = reinterpret_cast<const mma_u4 *>(at)[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = real && c + e < cols ? at[e] : S(0);
    }
}
struct StageJobs {
    StageJob job[4];
};
__global__ __launch_bounds__(256) void stage_kernel(StageJobs jobs) {
    const StageJob &j = jobs.job[blockIdx.y];
    const long pieces = j.pitch / 8, total = j.all * pieces;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long row = i / pieces;
        const int c = (int)(i % pieces) * 8;
        const long from = row < j.gate ? row : row < j.gate + j.move ? j.rows : row - j.move;
        const bool real = from < j.rows;
        uint16_t *to = j.dst + row * j.pitch + c;
        if (j.exps != nullptr) {
            const int8_t *at = reinterpret_cast<const int8_t *>(j.src) + from * j.cols + c;
            int8_t q[8];
            if (real && j.cols % 8 == 0) {
                *reinterpret_cast<mma_u2 *>(q) = *reinterpret_cast<const mma_u2 *>(at);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) q[e] = real && c + e < j.cols ? at[e] : (int8_t)0;
            }
            // (a group's eight values lie in it: groups are 32 wide)
            const float s = real && c < j.cols ? group_scale(j.exps[from * ((j.cols + kGroup8 - 1) / kGroup8) + c / kGroup8]) : 0.f;
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = c + e < j.cols ? (float)q[e] * s : 0.f;
            mma_u4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = pack16(j.type, v[2 * e], v[2 * e + 1]);
            *reinterpret_cast<mma_u4 *>(to) = w;
        } else if (j.type == DWO_F32) {
            float v[8], q[8][3];
            read_octet(reinterpret_cast<const float *>(j.src) + from * j.cols + c, c, j.cols, real, v);
#pragma unroll
            for (int e = 0; e < 8; e++) planes_of(v[e], q[e]);
#pragma unroll
            for (int k = 0; k < 3; k++)
                *reinterpret_cast<mma_u4 *>(to + k * j.plane) =
                    mma_u4{pack_bf16(q[0][k], q[1][k]), pack_bf16(q[2][k], q[3][k]), pack_bf16(q[4][k], q[5][k]),
                           pack_bf16(q[6][k], q[7][k])};
        } else {
            uint16_t v[8];
            read_octet(reinterpret_cast<const uint16_t *>(j.src) + from * j.cols + c, c, j.cols, real, v);
            *reinterpret_cast<mma_u4 *>(to) = *reinterpret_cast<const mma_u4 *>(v);
        }
    }
}

int Staging::launch(bool dry, hipStream_t st) {
    if (dry || count == 0) return 0;
    StageJobs all;
    long most = 0;
    for (int i = 0; i < count; i++) {
        all.job[i] = jobs[i];
        const long work = jobs[i].all * jobs[i].pitch / 8;
        most = work > most ? work : most;
    }
    stage_kernel<<<dim3(blocks_for(most, 8192), (unsigned)count), dim3(256), 0, st>>>(all);
    return status();
}

// Sums over the splits in a fixed order, then the plain epilogue: four neighbours of a row per thread, a product per blockIdx.y.
__global__ __launch_bounds__(256) void product_reduce_kernel(ProductGroup group) {
    const Product &p = group.part[blockIdx.y].p;
    const PlainEpi &epi = group.part[blockIdx.y].epi;
    if (epi.part == nullptr) return;
    const long quads = (p.N + 3) / 4, body = p.M * quads, all = body + (epi.sums.p != nullptr ? p.M : 0);
    const size_t total = (size_t)p.M * p.N;
    const float a = epi.scale();
    const bool four = p.N % 4 == 0;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long)gridDim.x * 256) {
        if (i >= body) {
            const long m = i - body, to = epi.place(m);
            const float *at = epi.part + p.splits * total + m;
            float v = 0.f;
#pragma unroll 4
            for (int s = 0; s < p.splits; s++) v += at[s * p.M];
            if (to >= 0) out_one(epi.sums, 0, to, v * a);
            continue;
        }
        const long m = i / quads, n = i % quads * 4, to = epi.place(m);
        const float *at = epi.part + (size_t)m * p.N + n;
        mma_f4 v = mma_f4{0.f, 0.f, 0.f, 0.f};
        if (four) {
#pragma unroll 4
            for (int s = 0; s < p.splits; s++) v += *reinterpret_cast<const mma_f4 *>(at + s * total);
        } else {
            for (int s = 0; s < p.splits; s++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (n + e < p.N) v[e] += at[s * total + e];
        }
        if (to < 0) continue;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (n + e < p.N) out_one(epi.out, to, n + e, epi.finish(to, n + e, v[e], a));
    }
}

template <typename T, class S>
__global__ __launch_bounds__(S::THREADS, S::PER_SIMD) void group_kernel(ProductGroup group) {
    DWO_STAGES(S);
    int block = (int)blockIdx.x, k = 0;
    while (k + 1 < group.count && block >= group.part[k].blocks) block -= group.part[k++].blocks;
    const GroupPart &q = group.part[k];
    switch (q.kind) {
        case 0: product_body<T, S, false, true, false>(q.p, q.epi, block, q.blocks, lds, nullptr); break;
        case 1: product_body<T, S, true, true, false>(q.p, q.epi, block, q.blocks, lds, nullptr); break;
        default: product_body<T, S, true, true, false>(q.p, SumsEpi{q.epi}, block, q.blocks, lds, nullptr);
    }
}

struct PlainChoice {
    int tile;
    long steps;  // of a split, at most
};
static long splits_for(long steps, long most) { return (steps + most - 1) / most; }

// When the last of the workgroups ends that go to 256 CUs one after the other, each to the CU that is free first, longest first:
// `count` kinds of them, numbers[i] of times[i]
static float makespan(const long *numbers, const float *times, int count) {
    struct Span {
        float end;
        long cus;
    } spans[16] = {{0.f, kLinCus}};
    int used = 1, order[3] = {0, 1, 2};
    for (int i = 1; i < count; i++)
        for (int k = i; k > 0 && times[order[k]] > times[order[k - 1]]; k--) std::swap(order[k], order[k - 1]);
    for (int i = 0; i < count; i++) {
        long n = numbers[order[i]];
        const float time = times[order[i]];
        // (of many only the last rounds are dealt out)
        if (n > 8 * kLinCus) {
            const long whole = n / kLinCus - 6;
            for (int k = 0; k < used; k++) spans[k].end += (float)whole * time;
            n -= whole * kLinCus;
        }
        while (n > 0) {
            int at = 0;
            for (int k = 1; k < used; k++)
                if (spans[k].end < spans[at].end) at = k;
            const long take = n < spans[at].cus ? n : spans[at].cus;
            const float end = spans[at].end + time;
            int same = 0;
            while (same < used && (same == at || spans[same].end != end)) same++;
            if (same == used && take == spans[at].cus) {
                spans[at].end = end;
            } else {
                if (same == used) {
                    if (used == 16) return end;
                    spans[used++] = {end, 0};
                }
                spans[same].cus += take, spans[at].cus -= take;
                if (spans[at].cus == 0) spans[at] = spans[--used];
            }
            n -= take;
        }
    }
    float last = 0.f;
    for (int k = 0; k < used; k++) last = spans[k].end > last ? spans[k].end : last;
    return last;
}

// The least of the products' time by tile_time's numbers, with splits of the sums also their writing and reading (4 TB/s behind each
// other) and the launch that joins them.  8192 x 1024 from 16384 and 16384 x 1024 from 8192, bf16: both in tiles of 256 without splits 430 us,
// the first one split in two, as it would be by itself, 470 and 33 for the join.
static PlainChoice find_choice(const GroupPart *part, int count) {
    PlainChoice best{0, 0};
    float least = 0.f;
    long longest = 0;
    for (int i = 0; i < count; i++) longest = part[i].p.steps > longest ? part[i].p.steps : longest;
    bool many = false;  // more than four workgroups a CU in the largest tiles
    for (const TileCost &c : kTileCosts) {
        bool chained = false;  // with fewer splits the longest sum takes more time than a CU's share of all
        for (const long parts : {1L, 2L, 3L, 4L, 6L, 8L, 12L, 16L, 24L, 32L}) {
            const long most = (longest + parts - 1) / parts;
            if (parts > 1 && most < 4) break;
            float join = 0.f, times[3];
            long workgroups = 0, chain = 0, numbers[3];
            for (int i = 0; i < count; i++) {
                const Product &p = part[i].p;
                const long splits = splits_for(p.steps, most), steps = (p.steps + splits - 1) / splits;
                numbers[i] = tiles_of(p.M, p.N, c.size, c.size) * splits, times[i] = c.more + (float)steps * c.more_step;
                workgroups += numbers[i];
                chain = steps > chain ? steps : chain;
                if (splits > 1) join += (float)(splits * p.M) * (float)p.N * 8.f / 4e6f + (join == 0.f ? 5.f : 0.f);
            }
            if (parts == 1 && c.size == kTileCosts[0].size) many = workgroups > 4 * kLinCus;
            // (one product may have that many without splits, and another's long sums be what is left to split: loss and gradients of 4 * 10^6 rows, 64
            // channels and 150 classes in bf16 3.2 ms, with that product in one piece 21; 10^6 x 32 x 16 0.45 and 2.55)
            if (parts > 1 && workgroups > 4 * kLinCus && !(many && chained)) break;
            if (c.size < kTileCosts[0].size && workgroups > kMostGroups - 8 * count) break;  // (each part's are rounded up to eight)
            const float alone = c.first + (float)chain * c.first_step;
            const float t = join + (workgroups <= kLinCus ? alone : fmaxf(alone, 3.5f + makespan(numbers, times, count)));
            float share = 0.f, most_time = 0.f;
            for (int i = 0; i < count; i++) share += (float)numbers[i] * times[i] / kLinCus, most_time = fmaxf(most_time, times[i]);
            chained = most_time > share;
            if (best.tile == 0 || t < least) best = {c.size, most}, least = t;
        }
    }
    return best;
}
// (a call asks three times for the same sizes, measuring its workspace and launching, and the next one often does: 64 answers are kept per
// thread, by all that they follow from)
static PlainChoice plain_choice(const GroupPart *part, int count) {
    struct Known {
        long key[9];
        PlainChoice choice;
    };
    static thread_local Known known[64] = {};
    long key[9] = {};
    size_t hash = 0;
    for (int i = 0; i < count; i++) {
        key[3 * i] = part[i].p.M, key[3 * i + 1] = part[i].p.N, key[3 * i + 2] = part[i].p.steps;
        for (int k = 0; k < 3; k++) hash = (hash ^ (size_t)key[3 * i + k]) * 0x9e3779b97f4a7c15ull, hash ^= hash >> 29;
    }
    Known &slot = known[hash % 64];
    bool same = slot.choice.tile != 0;
    for (int k = 0; k < 9; k++) same = same && slot.key[k] == key[k];
    if (!same) {
        for (int k = 0; k < 9; k++) slot.key[k] = key[k];
        slot.choice = find_choice(part, count);
    }
    return slot.choice;
}

static void split_part(GroupPart &q, const PlainChoice &choice, Arena &ws) {
    Product &p = q.p;
    const long splits = splits_for(p.steps, choice.steps);
    p.per = (int)((p.steps + splits - 1) / splits);
    p.splits = (p.steps + p.per - 1) / p.per;
    const size_t room = (size_t)p.splits * ((size_t)p.M * p.N + p.M) * sizeof(float);
    // (a workspace is measured for all outputs of a call: with some of them alone more splits may be chosen than it has room for)
    if (!ws.fits(room)) p.splits = 1, p.per = p.steps;
    q.epi.part = p.splits > 1 ? (float *)ws.take(room) : nullptr;
}
static int join_parts(const ProductGroup &group, hipStream_t st) {
    long work = 0;
    for (int i = 0; i < group.count; i++) {
        const Product &p = group.part[i].p;
        if (p.splits > 1 && p.M * ((p.N + 3) / 4) + p.M > work) work = p.M * ((p.N + 3) / 4) + p.M;
    }
    if (work == 0) return 0;
    product_reduce_kernel<<<dim3(blocks_for(work, 8192), (unsigned)group.count), dim3(256), 0, st>>>(group);
    return status();
}

template <typename T>
static int plain_typed(const GroupPart &q, int tile, hipStream_t st) {
    return with_tile<PlainEpi>(tile, tiles_of(q.p.M, q.p.N, tile, tile) * q.p.splits, q.p.per,
                     [&](auto shape) { return launch_shape<T, decltype(shape), false, false, false>(q.p, q.epi, st); });
}
int plain_product(const Operand &a, const Operand &b, long M, long N, long K, int dtype, PlainEpi epi, Arena &ws, hipStream_t st) {
    ProductGroup group;
    group.part[group.count++] = {make_product(a, b, M, N, K, 0), epi, 0, 0};
    const PlainChoice choice = plain_choice(group.part, 1);
    split_part(group.part[0], choice, ws);
    if (ws.dry()) return 0;
    const int e = dtype == DWO_F16 ? plain_typed<f16_t>(group.part[0], choice.tile, st) : plain_typed<bf16_t>(group.part[0], choice.tile, st);
    return e != 0 ? e : join_parts(group, st);
}

void ProductGroup::add(bool a_slow, const Operand &a, const Operand &b, long M, long N, long K, const PlainEpi &epi) {
    part[count++] = {make_product(a, b, M, N, K, 0), epi, !a_slow ? 0 : epi.sums.p == nullptr ? 1 : 2, 0};
}
template <typename T, class S>
static int launch_group(ProductGroup group, hipStream_t st) {
    long all = 0;
    for (int i = 0; i < group.count; i++) {
        Product &p = group.part[i].p;
        p.mtiles = (int)((p.M + S::BM - 1) / S::BM), p.ntiles = (int)((p.N + S::BN - 1) / S::BN);
        const long blocks = ((long)p.mtiles * p.ntiles * p.splits + 7) / 8 * 8;
        all += blocks;
        if (all > kMostGroups) return DWO_ERR_BAD_SHAPE;
        group.part[i].blocks = (int)blocks;
    }
    group_kernel<T, S><<<dim3((unsigned)all), dim3(S::THREADS), 0, st>>>(group);
    return status();
}
template <typename T>
static int launch_group_tile(const ProductGroup &group, int tile, hipStream_t st) {
    long workgroups = 0, steps = 0;
    for (int i = 0; i < group.count; i++) {
        const Product &p = group.part[i].p;
        workgroups += tiles_of(p.M, p.N, tile, tile) * p.splits;
        steps = p.per > steps ? p.per : steps;
    }
    return with_tile<PlainEpi>(tile, workgroups, steps, [&](auto shape) { return launch_group<T, decltype(shape)>(group, st); });
}
int ProductGroup::launch(int dtype, Arena &ws, hipStream_t st) {
    if (count == 0) return 0;
    const PlainChoice choice = plain_choice(part, count);
    for (int i = 0; i < count; i++) split_part(part[i], choice, ws);
    if (ws.dry()) return 0;
    // the longest sums first: what is left at the end is short
    for (int i = 1; i < count; i++)
        for (int k = i; k > 0 && part[k].p.per > part[k - 1].p.per; k--) std::swap(part[k], part[k - 1]);
    const int e = dtype == DWO_F16 ? launch_group_tile<f16_t>(*this, choice.tile, st) : launch_group_tile<bf16_t>(*this, choice.tile, st);
    return e != 0 ? e : join_parts(*this, st);
}

}  // namespace dwo
