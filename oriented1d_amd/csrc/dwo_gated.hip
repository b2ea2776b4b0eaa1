// The gated feed-forward block: a = x w_in^T + b_in = [g | u], h = act(g) u, y = h w_out^T + b_out, and its backward pass.
//
// Forward: both projections are one product whose tiles hold the gates of some hidden units and what these multiply side by
// side, so that h is made from the sums in registers; the second product reads it.  Backward: dh = dy w_out, and from its sums
// [dg | du] = [dh u act'(g) | dh act(g)] and h again, in registers; then dx = [dg du] w_in, dw_in = [dg du]^T x, dw_out = dy^T h.
//
// g and u are kept for the backward pass in fp32, eight bytes a hidden unit and row: what a composition of layers in 16 bits keeps as
// four tensors, without their roundings (dx would be 1.8 times a rounding off instead of 1.4).  Or nothing but x in 8 bits is kept, and the
// backward pass makes g and u again, into its workspace.  h, dg and du are rounded to the activations' type, as operands of the matrix cores,
// or to two of them where the work is small (kHalvesWork).
//
// 16384 x 1024 -> 4096 -> 1024 in bf16: the gated product 380 us and the one behind dy 335, bound by what goes out and comes in behind their
// sums (678 MB written; 537 MB read, 405 written: with the products' own reads 2.9 and 3.6 TB/s, matrix cores busy 29 and 15 %); the second
// product 135 (1018 TFLOP/s) and the group of the three gradients 680 (1010).  Tiles of 128, two workgroups a CU of which one writes while the
// other multiplies, take 474 and 341.  One row (dwo_few.h): 7.0 us, 25 MB of weights at 3.6 TB/s.
#include "dwo_check8.h"
#include "dwo_few.h"

namespace dwo {

struct GluEpi {
    static constexpr bool kSums = false, kDirect = false;
    Values bias;  // [2 H]
    long H, Hp;
    int act;
    float *keep;  // g, then u, [M][Hp] each; or null
    Out h;        // [M][Hp]; or p null
    struct Lane {
        float gate[8], up[8];
    };
    __device__ __forceinline__ Lane begin(const Product &, long n) const {
        Lane l;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const bool real = bias.p != nullptr && n + e < H;
            l.gate[e] = real ? bias.at(n + e) : 0.f, l.up[e] = real ? bias.at(H + n + e) : 0.f;
        }
        return l;
    }
    static constexpr int kRow = 0;
    __device__ __forceinline__ Nothing load(const Product &, long, long) const { return {}; }
    __device__ __forceinline__ void octet(const Product &p, const Lane &l, long m, long n, float (&g)[8], float (&u)[8]) const {
        if (m >= p.M || n >= Hp) return;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const bool real = n + e < H;
            g[e] = real ? g[e] + l.gate[e] : 0.f, u[e] = real ? u[e] + l.up[e] : 0.f;
        }
        if (keep != nullptr) {
            out_octet({keep, Hp, 0, OUT_F32}, true, m, n, Hp, g);
            out_octet({keep + p.M * Hp, Hp, 0, OUT_F32}, true, m, n, Hp, u);
        }
        if (h.p == nullptr) return;
#pragma unroll
        for (int e = 0; e < 8; e++) g[e] = act_value(act, g[e]) * u[e];
        operand_octet<false>(h, m, n, Hp, g);
    }
};

struct DgluEpi {
    static constexpr bool kSums = false, kDirect = false;
    long H, Hp;
    int act;
    const float *keep;
    Out dg, du, h;  // dg and du: two halves of one [M][2 Hp]
    static constexpr int kRow = 0;
    __device__ __forceinline__ Nothing begin(const Product &, long) const { return {}; }
    struct Data {
        mma_f4 gate[2], up[2];
    };
    __device__ __forceinline__ Data load(const Product &p, long m, long n) const {
        Data d;
        const mma_f4 *g = reinterpret_cast<const mma_f4 *>(keep + m * Hp + n);
        const mma_f4 *u = reinterpret_cast<const mma_f4 *>(keep + (p.M + m) * Hp + n);
        if (m < p.M && n < Hp)
            d = {{__builtin_nontemporal_load(g), __builtin_nontemporal_load(g + 1)},
                 {__builtin_nontemporal_load(u), __builtin_nontemporal_load(u + 1)}};
        return d;
    }
    __device__ __forceinline__ void octet(const Product &p, const Nothing &, const unsigned *, const Data &kept, int, long m, long n,
                                          float (&d)[8]) const {
        if (m >= p.M || n >= Hp) return;
        float a[8], b[8], o[8];
        const auto &[gate, up] = kept;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float value, slope;
            act_both(act, gate[e / 4][e % 4], value, slope);
            const bool real = n + e < H;
            const float v = up[e / 4][e % 4];
            a[e] = real ? d[e] * v * slope : 0.f, b[e] = real ? d[e] * value : 0.f, o[e] = real ? value * v : 0.f;
        }
        operand_octet(dg, m, n, Hp, a);
        operand_octet(du, m, n, Hp, b);
        operand_octet(h, m, n, Hp, o);
    }
};

struct GatedSizes {
    long rows, C, H, D, Hp;
    int dtype;
    GatedSizes(size_t r, int c, int h, int d, int t) : rows((long)r), C(c), H(h), D(d), Hp(up8(h)), dtype(t) {}
    double work() const { return (double)rows * (double)H * (double)(2 * C + D); }
    bool ok() const {
        return rows >= 1 && rows <= 1L << 30 && C >= 1 && H >= 1 && D >= 1 && C <= 65536 && H <= 65536 && D <= 65536 && known(dtype);
    }
};

static int gated_hidden(const GatedSizes &s, const Operand &x, const Operand &w, const void *b_in, int act, float *keep, const Out &h,
                        hipStream_t st) {
    const GluEpi epi{{b_in, s.dtype}, s.H, s.Hp, act, keep, h};
    // (the tile's columns are counted over both halves)
    return launch_product<false, false, true>(make_product(x, w, s.rows, 2 * s.H, s.C, s.H * w.pitch), s.dtype, epi, st);
}

static int gated_forward(const GatedSizes &s, const void *x, const void *w_in, const void *b_in, const void *w_out, const void *b_out,
                         void *y, float *keep, int act, Arena &ws, hipStream_t st) {
    if (few(s.rows, s.C, s.dtype) && few(s.rows, s.H, s.dtype)) {
        float *const h = (float *)ws.take((size_t)s.rows * s.H * sizeof(float));  // (few values: not rounded)
        if (ws.dry()) return 0;
        const FewGlu glu{{b_in, s.dtype}, s.rows, s.H, s.Hp, act, keep, h};
        const int e = launch_few<false>(x, w_in, s.C, s.H, s.H, s.rows, s.dtype, glu, st);
        return e != 0 ? e : launch_few<true>(h, w_out, s.H, s.D, 0, s.rows, s.dtype, FewPlain{{b_out, s.dtype}, {y, s.D, 0, s.dtype}}, st);
    }
    Staging stage;
    const Operand ox = stage.matrix(x, s.rows, s.C, s.dtype, ws), oi = stage.matrix(w_in, 2 * s.H, s.C, s.dtype, ws),
                  oo = stage.matrix(w_out, s.D, s.H, s.dtype, ws);
    int e = stage.launch(ws.dry(), st);
    if (e) return e;
    const Operand h = take_operand(ws, s.rows, s.Hp, s.dtype, s.work());
    if (!ws.dry() && (e = gated_hidden(s, ox, oi, b_in, act, keep, out_of(h, s.dtype), st))) return e;
    PlainEpi epi = plain_epilogue({y, s.D, 0, s.dtype});
    epi.bias = {b_out, s.dtype};
    return plain_product(h, oo, s.rows, s.D, s.H, s.dtype, epi, ws, st);
}

struct GatedGrads {
    void *dx, *dw_in, *db_in, *dw_out, *db_out;  // each may be null
    int grad;                                    // type of the parameters' gradients
};
// x, or its 8-bit form where keep is null
static int gated_backward(const GatedSizes &s, const void *dy, const void *x, const int8_t *codes, const uint8_t *exps, const float *keep,
                          const void *w_in, const void *b_in, const void *w_out, const GatedGrads &g, int act, Arena &ws,
                          hipStream_t st) {
    const long move = s.Hp - s.H;
    Staging stage;
    const Operand ody = stage.matrix(dy, s.rows, s.D, s.dtype, ws), oo = stage.matrix(w_out, s.D, s.H, s.dtype, ws),
                  oi = stage.matrix(w_in, 2 * s.H, s.C, s.dtype, ws, s.H, move);
    const Operand ox = codes != nullptr     ? stage.held8(codes, exps, s.rows, s.C, s.dtype, ws)
                       : g.dw_in != nullptr ? stage.matrix(x, s.rows, s.C, s.dtype, ws)
                                            : Operand{nullptr, 0, 0, 1};
    int e = stage.launch(ws.dry(), st);
    if (e) return e;
    if (keep == nullptr) {
        float *again = (float *)ws.take((size_t)2 * s.rows * s.Hp * sizeof(float));
        // (the rows of w_in's second half lie Hp rows behind the first's)
        const GluEpi epi{{b_in, s.dtype}, s.H, s.Hp, act, again, {nullptr, 0, 0, 0}};
        if (!ws.dry() &&
            (e = launch_product<false, false, true>(make_product(ox, oi, s.rows, 2 * s.H, s.C, s.Hp * oi.pitch), s.dtype, epi, st)))
            return e;
        keep = again;
    }
    const Operand da = take_operand(ws, s.rows, 2 * s.Hp, s.dtype, s.work()), h = take_operand(ws, s.rows, s.Hp, s.dtype, s.work());
    if (!ws.dry()) {
        const Out dg = out_of(da, s.dtype);
        Out du = dg;
        du.p = (uint16_t *)dg.p + s.Hp;
        const DgluEpi epi{s.H, s.Hp, act, keep, dg, du, out_of(h, s.dtype)};
        if ((e = launch_product<false, true, false>(make_product(ody, oo, s.rows, s.H, s.D, 0), s.dtype, epi, st))) return e;
    }
    ProductGroup group;
    if (g.dx != nullptr) group.add(false, da, oi, s.rows, s.C, 2 * s.Hp, plain_epilogue({g.dx, s.C, 0, s.dtype}));
    if (g.dw_in != nullptr) {
        PlainEpi epi = plain_epilogue({g.dw_in, s.C, 0, g.grad});
        epi.sums = {g.db_in, 0, 0, g.grad};
        epi.rows_from = s.Hp, epi.rows_skip = move, epi.tail = 2 * s.H;
        group.add(true, da, ox, 2 * s.Hp, s.C, s.rows, epi);
    }
    if (g.dw_out != nullptr) {
        PlainEpi epi = plain_epilogue({g.dw_out, s.H, 0, g.grad});
        epi.sums = {g.db_out, 0, 0, g.grad};
        group.add(true, ody, h, s.D, s.H, s.rows, epi);
    }
    return group.launch(s.dtype, ws, st);
}

}  // namespace dwo

using namespace dwo;

extern "C" {

size_t dwo_gated_workspace_bytes(size_t rows, int C, int H, int D, int backward, int held8, int dtype) {
    const GatedSizes s(rows, C, H, D, dtype);
    if (!s.ok()) return 0;
    Arena ws = Arena::measure();
    void *const any = (void *)256;  // (nothing is launched)
    if (!backward) {
        gated_forward(s, any, any, any, any, any, any, nullptr, ACT_GELU, ws, nullptr);
    } else {
        const GatedGrads g{any, any, any, any, any, DWO_F32};
        gated_backward(s, any, any, held8 ? (const int8_t *)any : nullptr, (const uint8_t *)any, held8 ? nullptr : (const float *)any,
                       any, any, any, g, ACT_GELU, ws, nullptr);
    }
    return ws.used + 256;
}

int dwo_gated_forward(const void *x, const void *w_in, const void *b_in, const void *w_out, const void *b_out, void *y, float *keep,
                      void *ws, size_t ws_bytes, size_t rows, int C, int H, int D, int act, int dtype, void *stream) {
    if (!x || !w_in || !w_out || !y || !ws) return DWO_ERR_NULL_POINTER;
    const GatedSizes s(rows, C, H, D, dtype);
    if (!known(dtype)) return DWO_ERR_BAD_DTYPE;
    if (!s.ok() || act < 0 || act > ACT_SILU ||
        ((uintptr_t)x | (uintptr_t)w_in | (uintptr_t)w_out | (uintptr_t)ws | (uintptr_t)keep) % 16 != 0)
        return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_gated_workspace_bytes(rows, C, H, D, 0, 0, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    Arena a{(char *)ws, 0, ws_bytes};
    return gated_forward(s, x, w_in, b_in, w_out, b_out, y, keep, act, a, (hipStream_t)stream);
}

int dwo_gated_backward(const void *dy, const void *x, const void *codes, const void *exps, const float *keep, const void *w_in,
                       const void *b_in, const void *w_out, void *dx, void *dw_in, void *db_in, void *dw_out, void *db_out, void *ws,
                       size_t ws_bytes, size_t rows, int C, int H, int D, int act, int dtype, int grad_dtype, void *stream) {
    const bool held8 = codes != nullptr;
    if (!dy || !w_in || !w_out || !ws || (held8 ? !exps || keep : !x || !keep)) return DWO_ERR_NULL_POINTER;
    const GatedSizes s(rows, C, H, D, dtype);
    if (!known(dtype) || !known(grad_dtype)) return DWO_ERR_BAD_DTYPE;
    if (!s.ok() || act < 0 || act > ACT_SILU || (db_in && !dw_in) || (db_out && !dw_out) ||
        ((uintptr_t)dy | (uintptr_t)x | (uintptr_t)w_in | (uintptr_t)w_out | (uintptr_t)ws | (uintptr_t)keep) % 16 != 0)
        return DWO_ERR_BAD_SHAPE;
    if (ws_bytes < dwo_gated_workspace_bytes(rows, C, H, D, 1, held8, dtype)) return DWO_ERR_SCRATCH_TOO_SMALL;
    (void)hipGetLastError();
    Arena a{(char *)ws, 0, ws_bytes};
    return gated_backward(s, dy, x, (const int8_t *)codes, (const uint8_t *)exps, keep, w_in, b_in, w_out,
                          {dx, dw_in, db_in, dw_out, db_out, grad_dtype}, act, a, (hipStream_t)stream);
}

}  // extern "C"
