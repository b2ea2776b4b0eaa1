// 8-bit checkpoints (dwo_check8.h): packing and unpacking, activations whose backward pass reads one, and layers whose weight
// gradients do.  Eight neighbours per lane, four lanes a group, sixteen bytes and more per access.  With GELU, 25088 x 1536 in bf16, both
// passes run at a large copy's rate and at the issue slots' at once: there 36 us (194 MB, 5.3 TB/s; 92 % of the slots), back 33 us (5.9 TB/s;
// 82 %).  A layer of 25088 x 384 -> 1536 packs its input in 7 us and stages it again in 9, of 150 both ways.
#include "dwo_check8.h"
#include "dwo_few.h"

namespace dwo {

// (elementwise passes: the activations' error is a fraction of their result's rounding)
template <typename T>
__device__ __forceinline__ void act_wide(int act, float g, float &value, float &slope) {
    if (act == ACT_SILU || sizeof(T) == 4) {
        act_both(act, g, value, slope);
    } else {
        value = gelu_rounded(g), slope = gelu_slope_rounded(g);
    }
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
    mma_u4 w[sizeof(T) / 2];
#pragma unroll
    for (int e = 0; e < (int)sizeof(T) / 2; e++) w[e] = reinterpret_cast<const mma_u4 *>(p)[e];
    const T *t = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = to_float(t[e]);
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<mma_f4 *>(p)[0] = mma_f4{v[0], v[1], v[2], v[3]};
        reinterpret_cast<mma_f4 *>(p)[1] = mma_f4{v[4], v[5], v[6], v[7]};
    } else {
        *reinterpret_cast<mma_u4 *>(p) = mma_u4{lin_pack<T>(v[0], v[1]), lin_pack<T>(v[2], v[3]), lin_pack<T>(v[4], v[5]),
                                                lin_pack<T>(v[6], v[7])};
    }
}
__device__ __forceinline__ void codes8(mma_u2 w, float (&q)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) q[e] = (float)((int)(w[e / 4] << (24 - 8 * (e % 4))) >> 24);
}

// Codes of x, where codes is not null, and where y is not null y = act(x).  WIDE: rows of whole groups, eight values per lane; otherwise half a
// wave takes a group, a value per lane.
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void pack8_kernel(const T *__restrict__ x, T *__restrict__ y, int8_t *__restrict__ codes,
                                                    uint8_t *__restrict__ exps, long rows, int C, int act) {
    const int groups = (C + kGroup8 - 1) / kGroup8;
    constexpr int LANES = WIDE ? 4 : 32;
    const long total = rows * groups * LANES;  // (a group's lanes stay together: 256 is a multiple of LANES)
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long group = i / LANES;
        if constexpr (WIDE) {
            float v[8];
            load8(x + i * 8, v);
            if (codes != nullptr) {
                unsigned most = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) most = max(most, magnitude(v[e]));
                most = max(most, (unsigned)__shfl_xor((int)most, 1, 64));
                most = max(most, (unsigned)__shfl_xor((int)most, 2, 64));
                const unsigned e = group_exponent(__uint_as_float(most));
                const float inverse = group_inverse(e);
                mma_u2 w = mma_u2{0u, 0u};
#pragma unroll
                for (int k = 0; k < 8; k++) w[k / 4] |= (unsigned)(quantum(v[k], inverse) & 0xff) << (8 * (k % 4));
                if (e == 255u) w = mma_u2{0u, 0u};
                reinterpret_cast<mma_u2 *>(codes)[i] = w;
                if (i % LANES == 0) exps[group] = (uint8_t)e;
            }
            if (y != nullptr) {
                float o[8], slope;
#pragma unroll
                for (int k = 0; k < 8; k++) act_wide<T>(act, v[k], o[k], slope);
                store8(y + i * 8, o);
            }
        } else {
            const long row = group / groups;
            const int c = (int)(group % groups) * kGroup8 + (int)(i % LANES);
            const bool real = c < C;
            const long at = row * C + c;
            const float v = real ? to_float(x[at]) : 0.f;
            if (codes != nullptr) {
                unsigned most = magnitude(v);
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) most = max(most, (unsigned)__shfl_xor((int)most, off, 64));
                const unsigned e = group_exponent(__uint_as_float(most));
                if (real) codes[at] = e == 255u ? 0 : (int8_t)quantum(v, group_inverse(e));
                if (i % LANES == 0) exps[group] = (uint8_t)e;
            }
            if (y != nullptr && real) {
                float o, slope;
                act_wide<T>(act, v, o, slope);
                y[at] = from_float<T>(o);
            }
        }
    }
}

// The values held, or where dy is not null dx = dy act'(value).
template <typename T, bool WIDE>
__global__ __launch_bounds__(256) void unpack8_kernel(const int8_t *__restrict__ codes, const uint8_t *__restrict__ exps,
                                                      const T *__restrict__ dy, T *__restrict__ out, long rows, int C,
                                                      int act) {
    const int groups = (C + kGroup8 - 1) / kGroup8;
    const long total = WIDE ? rows * C / 8 : rows * C;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        if constexpr (WIDE) {
            float v[8];
            codes8(reinterpret_cast<const mma_u2 *>(codes)[i], v);
            const float s = group_scale(exps[i / 4]);
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] *= s;
            if (dy != nullptr) {
                float d[8];
                load8(dy + i * 8, d);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    float value, slope;
                    act_wide<T>(act, v[e], value, slope);
                    v[e] = d[e] * slope;
                }
            }
            store8(out + i * 8, v);
        } else {
            const long row = i / C;
            const int c = (int)(i % C);
            float v = (float)codes[i] * group_scale(exps[row * groups + c / kGroup8]);
            if (dy != nullptr) {
                float value, slope;
                act_wide<T>(act, v, value, slope);
                v = to_float(dy[i]) * slope;
            }
            out[i] = from_float<T>(v);
        }
    }
}

template <typename T>
int launch_pack8(const void *x, void *y, void *codes, void *exps, long rows, int C, int act, hipStream_t st) {
    const bool wide = C % kGroup8 == 0;
    const long threads = rows * ((C + kGroup8 - 1) / kGroup8) * (wide ? 4 : 32);
    const dim3 grid(blocks_for(threads, 1 << 20)), block(256);
    if (wide) pack8_kernel<T, true><<<grid, block, 0, st>>>((const T *)x, (T *)y, (int8_t *)codes, (uint8_t *)exps, rows, C, act);
    else pack8_kernel<T, false><<<grid, block, 0, st>>>((const T *)x, (T *)y, (int8_t *)codes, (uint8_t *)exps, rows, C, act);
    return status();
}
template <typename T>
int launch_unpack8(const void *codes, const void *exps, const void *dy, void *out, long rows, int C, int act, hipStream_t st) {
    const bool wide = C % kGroup8 == 0;
    const dim3 grid(blocks_for(wide ? rows * C / 8 : rows * C, 1 << 20)), block(256);
    if (wide)
        unpack8_kernel<T, true><<<grid, block, 0, st>>>((const int8_t *)codes, (const uint8_t *)exps, (const T *)dy, (T *)out, rows, C,
                                                        act);
    else
        unpack8_kernel<T, false><<<grid, block, 0, st>>>((const int8_t *)codes, (const uint8_t *)exps, (const T *)dy, (T *)out, rows,
                                                         C, act);
    return status();
}

static bool sizes_ok(long rows, int C, const void *a, const void *b, const void *c, const void *d) {
    return rows >= 1 && rows <= 1L << 30 && C >= 1 && C <= 65536 && ((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) % 16 == 0;
}

static int layer_forward(const void *x, const void *w, const void *b, void *y, long rows, int C, int D, int dtype, Arena &ws,
                         hipStream_t st) {
    if (few(rows, C, dtype))
        return ws.dry() ? 0 : launch_few<false>(x, w, C, D, 0, rows, dtype, FewPlain{{b, dtype}, {y, D, 0, dtype}}, st);
    Staging stage;
    const Operand ox = stage.matrix(x, rows, C, dtype, ws), ow = stage.matrix(w, D, C, dtype, ws);
    const int e = stage.launch(ws.dry(), st);
    if (e) return e;
    PlainEpi epi = plain_epilogue({y, D, 0, dtype});
    epi.bias = {b, dtype};
    return plain_product(ox, ow, rows, D, C, dtype, epi, ws, st);
}
static int layer_backward(const void *dy, const int8_t *codes, const uint8_t *exps, const void *w, void *dx, void *dw, void *db,
                          long rows, int C, int D, int dtype, int grad, Arena &ws, hipStream_t st) {
    Staging stage;
    const Operand oy = stage.matrix(dy, rows, D, dtype, ws);
    const Operand ow = dx != nullptr ? stage.matrix(w, D, C, dtype, ws) : Operand{};
    const Operand ox = dw != nullptr ? stage.held8(codes, exps, rows, C, dtype, ws) : Operand{};
    const int e = stage.launch(ws.dry(), st);
    if (e) return e;
    ProductGroup group;
    if (dx != nullptr) group.add(false, oy, ow, rows, C, D, plain_epilogue({dx, C, 0, dtype}));
    if (dw != nullptr) {
        PlainEpi epi = plain_epilogue({dw, C, 0, grad});
        epi.sums = {db, 0, 0, grad};
        group.add(true, oy, ox, D, C, rows, epi);
    }
    return group.launch(dtype, ws, st);
}

}  // namespace dwo

using namespace dwo;

extern "C" {

int dwo_pack8(const void *x, void *y, void *codes, void *exps, size_t rows, int C, int act, int dtype, void *stream) {
    if (!x || (codes != nullptr ? !exps : !y)) return DWO_ERR_NULL_POINTER;
    if (!sizes_ok((long)rows, C, x, y, codes, nullptr) || act < 0 || act > ACT_SILU) return DWO_ERR_BAD_SHAPE;
    (void)hipGetLastError();
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case DWO_F32: return launch_pack8<float>(x, y, codes, exps, (long)rows, C, act, st);
        case DWO_BF16: return launch_pack8<bf16_t>(x, y, codes, exps, (long)rows, C, act, st);
        case DWO_F16: return launch_pack8<f16_t>(x, y, codes, exps, (long)rows, C, act, st);
        default: return DWO_ERR_BAD_DTYPE;
    }
}

int dwo_unpack8(const void *codes, const void *exps, const void *dy, void *out, size_t rows, int C, int act, int dtype, void *stream) {
    if (!codes || !exps || !out) return DWO_ERR_NULL_POINTER;
    if (!sizes_ok((long)rows, C, codes, dy, out, nullptr) || act < 0 || act > ACT_SILU) return DWO_ERR_BAD_SHAPE;
    (void)hipGetLastError();
    hipStream_t st = (hipStream_t)stream;
    switch (dtype) {
        case DWO_F32: return launch_unpack8<float>(codes, exps, dy, out, (long)rows, C, act, st);
        case DWO_BF16: return launch_unpack8<bf16_t>(codes, exps, dy, out, (long)rows, C, act, st);
        case DWO_F16: return launch_unpack8<f16_t>(codes, exps, dy, out, (long)rows, C, act, st);
        default: return DWO_ERR_BAD_DTYPE;
    }
}

size_t dwo_layer8_workspace_bytes(size_t rows, int C, int D, int backward, int dtype) {
    if (!sizes_ok((long)rows, C, nullptr, nullptr, nullptr, nullptr) || D < 1 || D > 65536 || !known(dtype)) return 0;
    Arena ws = Arena::measure();
    void *const any = (void *)256;  // (nothing is launched)
    if (backward)
        layer_backward(any, (const int8_t *)any, (const uint8_t *)any, any, any, any, any, (long)rows, C, D, dtype, DWO_F32, ws, nullptr);
    else
        layer_forward(any, any, any, any, (long)rows, C, D, dtype, ws, nullptr);
    return ws.used + 256;
}

int dwo_layer8(const void *x, const void *w, const void *bias, void *y, void *codes, void *exps, void *ws, size_t ws_bytes, size_t rows,
               int C, int D, int dtype, void *stream) {
    if (!x || !w || !y || !ws || (codes != nullptr && !exps)) return DWO_ERR_NULL_POINTER;
    if (!known(dtype)) return DWO_ERR_BAD_DTYPE;
    if (!sizes_ok((long)rows, C, x, w, ws, codes) || D < 1 || D > 65536) return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_layer8_workspace_bytes(rows, C, D, 0, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    if (codes != nullptr) {
        const int e = dwo_pack8(x, nullptr, codes, exps, rows, C, 0, dtype, stream);
        if (e != 0) return e;
    }
    Arena a{(char *)ws, 0, ws_bytes};
    return layer_forward(x, w, bias, y, (long)rows, C, D, dtype, a, (hipStream_t)stream);
}

int dwo_layer8_backward(const void *dy, const void *codes, const void *exps, const void *w, void *dx, void *dw, void *db, void *ws,
                        size_t ws_bytes, size_t rows, int C, int D, int dtype, int grad_dtype, void *stream) {
    if (!dy || !codes || !exps || !w || !ws) return DWO_ERR_NULL_POINTER;
    if (!known(dtype) || !known(grad_dtype)) return DWO_ERR_BAD_DTYPE;
    if (!sizes_ok((long)rows, C, dy, w, ws, codes) || D < 1 || D > 65536 || (db && !dw)) return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_layer8_workspace_bytes(rows, C, D, 1, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    Arena a{(char *)ws, 0, ws_bytes};
    return layer_backward(dy, (const int8_t *)codes, (const uint8_t *)exps, w, dx, dw, db, (long)rows, C, D, dtype, grad_dtype, a,
                          (hipStream_t)stream);
}

}  // extern "C"
