// Operands of the products around wide layers, and the products with the plain epilogue.
#include "dwo_product.h"

namespace dwo {

// rows x cols of a dense matrix as an operand: columns padded with zeros to `pitch`, fp32 taken apart into three planes.  Rows from
// `gate` on go `move` rows further down (the second half of gated weights whose hidden size is no multiple of eight), the rest is zeros.
template <typename S>
__global__ __launch_bounds__(256) void stage_kernel(const S *__restrict__ src, uint16_t *__restrict__ dst, long rows, int cols,
                                                    long gate, long move, long all_rows, long pitch, long plane) {
    const long pieces = pitch / 8, total = all_rows * pieces;
    const bool wide = cols % (16 / (int)sizeof(S)) == 0;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long row = i / pieces;
        const int c = (int)(i % pieces) * 8;
        const long from = row < gate ? row : row < gate + move ? rows : row - move;
        const S *at = src + from * cols + c;
        S v[8];
        if (from < rows && wide && c + 8 <= cols) {
#pragma unroll
            for (int e = 0; e < (int)sizeof(S) / 2; e++)
                reinterpret_cast<mma_u4 *>(v)[e] = reinterpret_cast<const mma_u4 *>(at)[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = from < rows && c + e < cols ? at[e] : S(0);
        }
        uint16_t *to = dst + row * pitch + c;
        if constexpr (sizeof(S) == 4) {
            float q[8][3];
#pragma unroll
            for (int e = 0; e < 8; e++) planes_of(v[e], q[e]);
#pragma unroll
            for (int k = 0; k < 3; k++)
                *reinterpret_cast<mma_u4 *>(to + k * plane) =
                    mma_u4{pack_bf16(q[0][k], q[1][k]), pack_bf16(q[2][k], q[3][k]), pack_bf16(q[4][k], q[5][k]),
                           pack_bf16(q[6][k], q[7][k])};
        } else {
            *reinterpret_cast<mma_u4 *>(to) = *reinterpret_cast<const mma_u4 *>(v);
        }
    }
}

int stage_operand(Operand &o, const void *src, long rows, long cols, int dtype, Arena &ws, hipStream_t st, long gate, long move) {
    if (dtype != DWO_F32 && cols % 8 == 0 && move == 0) {
        o = {src, cols, 0, 1};
        return 0;
    }
    const long all = rows + 2 * move;
    if (move == 0) gate = rows;
    o = take_operand(ws, all, up8(cols), dtype);
    if (ws.dry()) return 0;
    const dim3 grid(blocks_for(all * o.pitch / 8, 16384)), block(256);
    uint16_t *to = (uint16_t *)const_cast<void *>(o.p);
    if (dtype == DWO_F32)
        stage_kernel<float><<<grid, block, 0, st>>>((const float *)src, to, rows, (int)cols, gate, move, all, o.pitch, o.plane);
    else
        stage_kernel<uint16_t><<<grid, block, 0, st>>>((const uint16_t *)src, to, rows, (int)cols, gate, move, all, o.pitch, o.plane);
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
    return plain_shape<T, SmallTile>(p, as, bs, epi, st);
}

int plain_product(const Operand &a, bool as, const Operand &b, bool bs, long M, long N, long K, int dtype, PlainEpi epi, Arena &ws,
                  hipStream_t st) {
    Product p = make_product(a, b, M, N, K, 0);
    const long large = tiles_of(M, N, 256, 256), medium = tiles_of(M, N, 128, 128), small = tiles_of(M, N, 64, 64);
    const int tile = large >= 200 ? 256 : medium >= 160 || (medium >= 8 && p.steps >= 64) ? 128 : 64;
    const long tiles = tile == 256 ? large : tile == 128 ? medium : small;
    // as many splits as the chip holds workgroups, of eight steps at least
    const long room = tile == 256 ? 1 : (tile == 128 ? 512 : 1024) / tiles;
    long splits = p.steps / 8 < room ? p.steps / 8 : room;
    if (splits < 1) splits = 1;
    p.per = (int)((p.steps + splits - 1) / splits);
    p.splits = (p.steps + p.per - 1) / p.per;
    if (p.splits > 1) epi.part = (float *)ws.take((size_t)p.splits * ((size_t)M * N + M) * sizeof(float));
    if (ws.dry()) return 0;
    const int e = dtype == DWO_F16 ? plain_typed<f16_t>(p, tile, as, bs, epi, st) : plain_typed<bf16_t>(p, tile, as, bs, epi, st);
    if (e != 0 || p.splits == 1) return e;
    product_reduce_kernel<<<dim3(blocks_for(M * ((N + 3) / 4) + M, 8192)), dim3(256), 0, st>>>(p, epi);
    return status();
}

}  // namespace dwo
