// tz_act.cuh -- the activations of the gated feed-forward kernels and their derivatives, in f32.
#pragma once
#include "../../include/tenzor_cuda.h"

namespace tz {

__host__ __device__ __forceinline__ bool gated_act_ok(int act) {
    return act == TZ_OP_SILU || act == TZ_OP_GELU || act == TZ_OP_GELU_ERF || act == TZ_OP_RELU || act == TZ_OP_SIGMOID;
}

// 1 / (1 + e^-z) by the fast exponential and the approximate reciprocal (about 2^-21 relative; e^-z = inf
// gives 0).  tanh.approx would halve the special-function work but is only good to 2^-11, which an f16
// result would show.
__device__ __forceinline__ float sigmoid_fast(float z) { return __fdividef(1.0f, 1.0f + __expf(-z)); }

// act(g); with GRAD also act'(g) in `d`.  A NaN stays NaN in every form.
template <int ACT, bool GRAD>
__device__ __forceinline__ float gated_act(float g, float& d) {
    if constexpr (ACT == TZ_OP_SILU) {
        const float s = sigmoid_fast(g);
        const float a = g * s;
        if constexpr (GRAD) d = fmaf(a, 1.0f - s, s);  // s (1 + g (1 - s))
        return a;
    } else if constexpr (ACT == TZ_OP_GELU) {
        // 0.5 g (1 + tanh z) = g sigmoid(2 z), z = sqrt(2 / pi) (g + 0.044715 g^3)
        const float g2 = g * g;
        const float s = sigmoid_fast(1.5957691216057308f * g * fmaf(0.044715f, g2, 1.0f));
        if constexpr (GRAD) {
            // s + g s (1 - s) 2 z'; for large |g| the product s (1 - s) is 0 while z' overflows
            const float t = s * (1.0f - s);
            const float dz = 1.5957691216057308f * fmaf(0.134145f, g2, 1.0f);
            d = t == 0.0f ? s : fmaf(g * t, dz, s);
        }
        return g * s;
    } else if constexpr (ACT == TZ_OP_GELU_ERF) {
        const float c = 0.5f * (1.0f + erff(0.7071067811865476f * g));
        if constexpr (GRAD) d = fmaf(g * 0.3989422804014327f, __expf(-0.5f * g * g), c);
        return g * c;
    } else if constexpr (ACT == TZ_OP_RELU) {
        if constexpr (GRAD) d = g > 0.0f ? 1.0f : (g != g ? g : 0.0f);
        return g < 0.0f ? 0.0f : g;
    } else {
        const float s = sigmoid_fast(g);
        if constexpr (GRAD) d = s * (1.0f - s);
        return s;
    }
}

}  // namespace tz
