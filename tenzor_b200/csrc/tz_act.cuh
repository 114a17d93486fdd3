// tz_act.cuh -- the activations of the gated feed-forward kernels and their derivatives, in f32, two
// neighbouring values at a time (packed f32x2 arithmetic: one issue slot for two operations).
//
// What bounds them: the special-function unit takes 16 lanes a clock per SM and every smooth activation needs
// an exponential and a reciprocal, 2048 clocks for the 128 x 128 outputs of one tile and CTA; the packed
// arithmetic keeps the issue slots (about 6 per value) below that.
#pragma once
#include "../../include/tenzor_cuda.h"
#include "tz_ptx.cuh"

namespace tz {

__host__ __device__ __forceinline__ bool gated_act_ok(int act) {
    return act == TZ_OP_SILU || act == TZ_OP_GELU || act == TZ_OP_GELU_ERF || act == TZ_OP_RELU || act == TZ_OP_SIGMOID;
}

__device__ __forceinline__ uint64_t f2_all(float v) { return tzp::f2_pack(v, v); }

__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 1 / (1 + 2^z) of a pair, by the special-function unit (about 2^-21 relative; 2^z = inf gives 0).
// tanh.approx would halve the special-function work but is only good to 2^-11, which an f16 result would show.
__device__ __forceinline__ uint64_t logistic2(uint64_t z) {
    const float2 v = tzp::f2_unpack(z);
    const float2 d = tzp::f2_unpack(tzp::f2_add(tzp::f2_pack(tzp::ex2_approx(v.x), tzp::ex2_approx(v.y)), f2_all(1.0f)));
    return tzp::f2_pack(rcp_approx(d.x), rcp_approx(d.y));
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kGelu = 1.5957691216057308f;  // 2 sqrt(2 / pi): 0.5 g (1 + tanh z) = g sigmoid(2 z)

// act of a pair; with GRAD also act' in `d`.  A NaN stays NaN, and in its own place, in every form.
template <int ACT, bool GRAD>
__device__ __forceinline__ uint64_t gated_act2(uint64_t g, uint64_t& d) {
    using namespace tzp;
    if constexpr (ACT == TZ_OP_SILU) {
        const uint64_t s = logistic2(f2_mul(g, f2_all(-kLog2e)));
        const uint64_t a = f2_mul(g, s);
        if constexpr (GRAD) d = f2_fma(a, f2_sub(f2_all(1.0f), s), s);  // s (1 + g (1 - s))
        return a;
    } else if constexpr (ACT == TZ_OP_GELU) {
        uint64_t g2 = f2_mul(g, g);
        if constexpr (GRAD) {  // keeps 0 * inf out of the derivative; past 1e15 the logistic is 0 or 1 anyway
            const float2 q = f2_unpack(g2);
            g2 = f2_pack(fminf(q.x, 1e30f), fminf(q.y, 1e30f));
        }
        const uint64_t s = logistic2(f2_mul(g, f2_fma(g2, f2_all(-kLog2e * kGelu * 0.044715f), f2_all(-kLog2e * kGelu))));
        const uint64_t a = f2_mul(g, s);
        if constexpr (GRAD)  // s + g s (1 - s) (2 z)'
            d = f2_fma(f2_mul(a, f2_sub(f2_all(1.0f), s)), f2_fma(g2, f2_all(kGelu * 0.134145f), f2_all(kGelu)), s);
        return a;
    } else if constexpr (ACT == TZ_OP_GELU_ERF) {
        const float2 v = f2_unpack(g);
        const uint64_t c = f2_fma(f2_pack(erff(0.7071067811865476f * v.x), erff(0.7071067811865476f * v.y)), f2_all(0.5f), f2_all(0.5f));
        if constexpr (GRAD) {
            const float2 q = f2_unpack(f2_mul(f2_mul(g, g), f2_all(-0.5f * kLog2e)));
            d = f2_fma(f2_mul(g, f2_all(0.3989422804014327f)), f2_pack(ex2_approx(q.x), ex2_approx(q.y)), c);
        }
        return f2_mul(g, c);
    } else if constexpr (ACT == TZ_OP_RELU) {
        const float2 v = f2_unpack(g);
        if constexpr (GRAD) d = f2_pack(v.x > 0.0f ? 1.0f : (v.x != v.x ? v.x : 0.0f), v.y > 0.0f ? 1.0f : (v.y != v.y ? v.y : 0.0f));
        return f2_pack(v.x < 0.0f ? 0.0f : v.x, v.y < 0.0f ? 0.0f : v.y);
    } else {
        const uint64_t s = logistic2(f2_mul(g, f2_all(-kLog2e)));
        if constexpr (GRAD) d = f2_mul(s, f2_sub(f2_all(1.0f), s));
        return s;
    }
}

// Two gate / up pairs (f32 bits) to one packed 16-bit pair of outputs.
template <int ACT, bool BF>
__device__ __forceinline__ uint32_t gated_pair(uint32_t g0, uint32_t g1, uint32_t u0, uint32_t u1) {
    uint64_t d;
    const uint64_t a = gated_act2<ACT, false>(tzp::f2_pack(__uint_as_float(g0), __uint_as_float(g1)), d);
    const float2 h = tzp::f2_unpack(tzp::f2_mul(a, tzp::f2_pack(__uint_as_float(u0), __uint_as_float(u1))));
    return tzp::pack16x2<BF>(h.x, h.y);
}

// Two gate / up pairs and their outputs' gradients to packed 16-bit dg = dh u act'(g) and du = dh act(g).
template <int ACT, bool BF>
__device__ __forceinline__ void gated_pair_grad(uint32_t g0, uint32_t g1, uint32_t u0, uint32_t u1, float2 dh, uint32_t& dg, uint32_t& du) {
    uint64_t d;
    const uint64_t h2 = tzp::f2_pack(dh.x, dh.y);
    const uint64_t a = gated_act2<ACT, true>(tzp::f2_pack(__uint_as_float(g0), __uint_as_float(g1)), d);
    const float2 p = tzp::f2_unpack(tzp::f2_mul(tzp::f2_mul(h2, tzp::f2_pack(__uint_as_float(u0), __uint_as_float(u1))), d));
    const float2 q = tzp::f2_unpack(tzp::f2_mul(h2, a));
    dg = tzp::pack16x2<BF>(p.x, p.y);
    du = tzp::pack16x2<BF>(q.x, q.y);
}

#define TZ_ACT_SWITCH(act, CALL)                          \
    switch (act) {                                        \
        case TZ_OP_SILU: CALL(TZ_OP_SILU); break;         \
        case TZ_OP_GELU: CALL(TZ_OP_GELU); break;         \
        case TZ_OP_GELU_ERF: CALL(TZ_OP_GELU_ERF); break; \
        case TZ_OP_RELU: CALL(TZ_OP_RELU); break;         \
        default: CALL(TZ_OP_SIGMOID); break;              \
    }

}  // namespace tz
