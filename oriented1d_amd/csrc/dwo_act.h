// Activations with their slopes, in fp32.
#pragma once

#include "dwo_product.h"

namespace dwo {

enum { ACT_GELU = DWO_GELU, ACT_SILU = DWO_SILU };

// act(g), and with its slope, for sums that nothing has rounded.
//   GELU: g Phi(g), Phi + g phi, Phi from lin_gelu's polynomial (5.4e-8 off at most)
//   SiLU: g s, s (1 + g (1 - s)) with s = 1 / (1 + exp(-g))
__device__ __forceinline__ float act_value(int act, float g) {
    if (act == ACT_SILU) return g * __builtin_amdgcn_rcpf(1.f + prod_exp(-g));
    return lin_gelu(g);
}
__device__ __forceinline__ void act_both(int act, float g, float &value, float &slope) {
    if (act == ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + prod_exp(-g));
        value = g * s, slope = s * __builtin_fmaf(g, 1.f - s, 1.f);
        return;
    }
    const float t = __builtin_fabsf(g), half = lin_half_erf(t);
    value = __builtin_fmaf(t, half, 0.5f * g);
    slope = __builtin_fmaf(g * 0.398942280f, prod_exp(-0.5f * g * g), 0.5f + __builtin_copysignf(half, g));
}

}  // namespace dwo
