// The activations of a dense layer's epilogue and their slopes, in float32.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/gcn_hip.h"

namespace gcn {

// The normal distribution's tail Phi(-|z|) = erfc(x) / 2: erfc(x) = e^(-x^2) t P(t) with t = 1 / (1 + 0.4 x), x = |z| / sqrt(2).  P is a least-squares fit
// of degree 8 on x in [0, 13], reweighted towards the smallest largest relative error: 9e-8 of erfc itself everywhere, 2.5e-7
// with float32 arithmetic, so that the far tails keep their digits.  `e` returns e^(-z^2 / 2), the factor the normal
// density shares with it.  17 instructions; the library's erff takes about 50 in two branches.
__device__ __forceinline__ float normal_tail(float z, float* e) {
    const float a = fabsf(z);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.28284271247461903f, a, 1.0f));
    float p = 0.04596841707825661f;      // the last digits chosen so that P(1) is 1 exactly: Phi(0) = 1/2
    p = fmaf(p, t, -0.16306036710739136f);
    p = fmaf(p, t, 0.13050033152103424f);
    p = fmaf(p, t, 0.035431280732154846f);
    p = fmaf(p, t, 0.11547110229730606f);
    p = fmaf(p, t, 0.17847903072834015f);
    p = fmaf(p, t, 0.20561064779758453f);
    p = fmaf(p, t, 0.22593672573566437f);
    p = fmaf(p, t, 0.22566290199756622f);
    *e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
    return 0.5f * t * p * *e;
}

// act(z); a NaN stays one
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
    if (ACT == GCN_ACT_RELU) return z <= 0.0f ? 0.0f : z;
    if (ACT == GCN_ACT_GELU) {
        float e;
        const float tail = normal_tail(z, &e);
        return z * (z < 0.0f ? tail : 1.0f - tail);
    }
    if (ACT == GCN_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
    return z;
}

// act'(z)
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
    if (ACT == GCN_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
    if (ACT == GCN_ACT_GELU) {
        float e;
        const float tail = normal_tail(z, &e);
        return fmaf(z * 0.3989422804014327f, e, z < 0.0f ? tail : 1.0f - tail);
    }
    if (ACT == GCN_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f));
        return s * fmaf(z, 1.0f - s, 1.0f);
    }
    return 1.0f;
}

// calls f with the activation as a compile-time constant
template <class F>
__device__ __forceinline__ void with_act(int act, F f) {
    if (act == GCN_ACT_RELU) f(std::integral_constant<int, GCN_ACT_RELU>{});
    else if (act == GCN_ACT_GELU) f(std::integral_constant<int, GCN_ACT_GELU>{});
    else if (act == GCN_ACT_SILU) f(std::integral_constant<int, GCN_ACT_SILU>{});
    else f(std::integral_constant<int, GCN_ACT_NONE>{});
}

// The epilogue of a dense layer: C = act(A . B + bias) + residual, the pre-activation A . B + bias kept in pre.
struct EpiArgs {
    const float* bias;       // [n], may be null
    const float* residual;   // [m x n], may be null; may be C itself: the lane that stores an element has read it
    int64_t ldr;
    float* pre;              // [m x n], may be null
    int64_t ldp;
    int act;
};

// C = the epilogue of the sum of part [splits][m x n] (layer_grad.hip)
int launch_join_splits(int64_t m, int64_t n, int64_t splits, const float* part, const EpiArgs& ep, float* c, int64_t ldc,
                       hipStream_t st);

}  // namespace gcn
