// Operands of the products around wide layers, and the products with the plain epilogue.
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

// Sums over the splits in a fixed order, then the plain epilogue: four neighbours of a row per thread.
__global__ __launch_bounds__(256) void product_reduce_kernel(Product p, PlainEpi epi) {
    const long quads = (p.N + 3) / 4, body = p.M * quads, all = body + (epi.sums.p != nullptr ? p.M : 0);
    const size_t total = (size_t)p.M * p.N;
    const float a = epi.alpha != nullptr ? *epi.alpha : 1.f;
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
int plain_shape(const Product &p, bool as, bool bs, const PlainEpi &epi, hipStream_t st) {
    if (as && epi.sums.p != nullptr) return launch_shape<T, S, true, true, false>(p, SumsEpi{epi}, st);
    if (as) return launch_shape<T, S, true, true, false>(p, epi, st);
    if (bs) return launch_shape<T, S, false, true, false>(p, epi, st);
    return launch_shape<T, S, false, false, false>(p, epi, st);
}
template <typename T>
int plain_typed(const Product &p, int tile, bool as, bool bs, const PlainEpi &epi, hipStream_t st) {
    if (tile == 256) return plain_shape<T, LargeTile>(p, as, bs, epi, st);
    if (tile == 128) return plain_shape<T, MediumTile>(p, as, bs, epi, st);
    if (tile == 64) return plain_shape<T, SmallTile>(p, as, bs, epi, st);
    return plain_shape<T, ThinTile>(p, as, bs, epi, st);
}

// tile and splits of a plain product
struct PlainChoice {
    int tile;
    long splits;
};
// The least of tile_time, with splits of the sums their writing and reading (4 TB/s behind each other) and the launch that joins them
PlainChoice plain_choice(long M, long N, int steps) {
    PlainChoice best{0, 0};
    float least = 0.f;
    for (const TileCost &c : kTileCosts) {
        const long tiles = tiles_of(M, N, c.size, c.size);
        for (const long splits : {1L, 2L, 3L, 4L, 6L, 8L, 12L, 16L, 24L, 32L}) {
            if (splits > 1 && (tiles * splits > 4 * kLinCus || steps < 4 * splits)) break;
            float t = tile_time(c, tiles * splits, (steps + splits - 1) / splits);
            if (splits > 1) t += 4.f + (float)(splits * M) * (float)N * 8.f / 4e6f;
            if (best.tile == 0 || t < least) best = {c.size, splits}, least = t;
        }
    }
    return best;
}

int plain_product_as(Product p, const PlainChoice &choice, bool as, bool bs, int dtype, PlainEpi epi, Arena &ws, hipStream_t st) {
    p.per = (int)((p.steps + choice.splits - 1) / choice.splits);
    p.splits = (p.steps + p.per - 1) / p.per;
    if (p.splits > 1) epi.part = (float *)ws.take((size_t)p.splits * ((size_t)p.M * p.N + p.M) * sizeof(float));
    if (ws.dry()) return 0;
    const int e = dtype == DWO_F16 ? plain_typed<f16_t>(p, choice.tile, as, bs, epi, st) : plain_typed<bf16_t>(p, choice.tile, as, bs, epi, st);
    if (e != 0 || p.splits == 1) return e;
    product_reduce_kernel<<<dim3(blocks_for(p.M * ((p.N + 3) / 4) + p.M, 8192)), dim3(256), 0, st>>>(p, epi);
    return status();
}
int plain_product(const Operand &a, bool as, const Operand &b, bool bs, long M, long N, long K, int dtype, PlainEpi epi, Arena &ws,
                  hipStream_t st) {
    const Product p = make_product(a, b, M, N, K, 0);
    return plain_product_as(p, plain_choice(M, N, p.steps), as, bs, dtype, epi, ws, st);
}

}  // namespace dwo
