// The activations of the gated projections and the linears with an epilogue (gated.hip, gated_tiles.hip).
#pragma once
#include "node_tile.h"

namespace tgt {
namespace {

// 1 / (1 + exp(-u)).  EXACT (float32 results): exp2 of the product u log2(e) in two parts, so that its rounding does not grow with u, and one Newton step on the
// reciprocal (from 2^100 on, where the step would make NaNs of infinities, it is zero): fourteen instructions where expf and a division take forty.  Else the
// hardware's exp2 and reciprocal as they are, good to 2^-22 and |u| 2^-24: nothing of a result of 8 bits.
template <bool EXACT> __device__ __forceinline__ float sigmoid_of(float u) {
    constexpr float kLog2e = 1.4426950408889634f;
    const float hi = u * -kLog2e;
    if (!EXACT) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(hi));
    const float lo = fmaf(u, -kLog2e, -hi) + u * -1.925963033500e-8f;      // (log2(e) behind its 24 bits)
    float e = __builtin_amdgcn_exp2f(hi);
    e = fmaf(e * lo, 0.6931471805599453f, e);
    const float d = 1.f + e, r = __builtin_amdgcn_rcpf(d);
    const float s = fmaf(fmaf(-d, r, 1.f), r, r);
    return e < 0x1p100f ? s : (u == u ? 0.f : u);
}
// act(u), and dh * act'(u).  GELU with the distribution function of node_tile.h: a third of erff's instructions, no larger errors
template <bool EXACT, int ACT> __device__ __forceinline__ float act_of(float u) {
    if (ACT == TGT_ACT_SILU) return u * sigmoid_of<EXACT>(u);
    if (ACT == TGT_ACT_GELU) {
        float cdf, bell;
        normal_cdf(u, cdf, bell);
        return u * cdf;
    }
    if (ACT == TGT_ACT_RELU) return act_value<true>(u);
    return u;
}
template <bool EXACT, int ACT> __device__ __forceinline__ float slope_of(float u, float dh) {
    if (ACT == TGT_ACT_SILU) {
        const float s = sigmoid_of<EXACT>(u);
        return dh * (s * (1.f + u * (1.f - s)));
    }
    if (ACT == TGT_ACT_GELU) {
        float cdf, bell;
        normal_cdf(u, cdf, bell);
        return dh * fmaf(u * bell, 0.39894228040143268f, cdf);
    }
    if (ACT == TGT_ACT_RELU) return act_grad<true>(u, dh);
    return dh;
}

// Both at once: a = act(u), s = act'(u)
template <bool EXACT, int ACT> __device__ __forceinline__ void act_and_slope(float u, float& a, float& s) {
    if (ACT == TGT_ACT_SILU) {
        const float t = sigmoid_of<EXACT>(u);
        a = u * t;
        s = t * (1.f + u * (1.f - t));
    } else if (ACT == TGT_ACT_GELU) {
        float cdf, bell;
        normal_cdf(u, cdf, bell);
        a = u * cdf;
        s = fmaf(u * bell, 0.39894228040143268f, cdf);
    } else {
        a = act_of<EXACT, ACT>(u);
        s = slope_of<EXACT, ACT>(u, 1.f);
    }
}

}  // namespace
}  // namespace tgt
