// The gated feed-forward block's activations and their derivatives, float32.
#pragma once

#include "common.cuh"

namespace sffn {

enum { GLU_RELU = 0, GLU_RELU2 = 1, GLU_SILU = 2, GLU_GELU = 3 };

// Two float32 values, for the packed instructions: half the issue slots, which
// bound the fused epilogues (35 instructions an element before).
using Float2 = unsigned long long;
__device__ __forceinline__ Float2 join2(float lo, float hi) {
    Float2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 split2(Float2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ Float2 pair_mul(Float2 a, Float2 b) {
    Float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Float2 pair_add(Float2 a, Float2 b) {
    Float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Float2 pair_fma(Float2 a, Float2 b, Float2 c) {
    Float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {  // 2^x within 2 ulp; subnormals are 0
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {  // 1 / x within 1 ulp
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// act(g) and act'(g) of two elements.  SiLU: s = 1 / (1 + 2^(-g log2 e)) by the
// hardware's exp2 and reciprocal, within 2^-21 max(|g|, 2) of the value for g >= -92:
// below a tenth of a 16-bit rounding down to the smallest normal results.  (Exponential,
// sum and reciprocal are held 2^8 apart from their values: the reciprocal of a sum
// above 2^126 is flushed to 0, and at g = -88 it is s that is so small, not g s.  Below
// -92 the result may be 0.  Forward of 32768 x 768 x 2048: 287 us without, 288 with.)
// GELU is the exact one: Phi(-|g|) = e^(-g^2 / 2)
// t Q(t) with t = 1 / (1 + 0.2333 |g|), Q of degree 7 fitted here for the least relative
// error over all t (9.4e-8), so that small tails keep their digits: within 2.7e-6 of
// Phi for |g| < 5 in float32, 1.3e-5 at 12, where the exponent's rounding grows.
// (erfcf, element by element: 247 us for UP of 32768 x 768 x 2048.)
template <int ACT, bool GRAD>
__device__ __forceinline__ Float2 glu_act2(Float2 g, Float2& d) {
    if constexpr (ACT == GLU_SILU) {
        constexpr float low = 1.f / 256;
        const float2 t = split2(pair_fma(g, join2(-1.4426950408889634f, -1.4426950408889634f), join2(-8.f, -8.f)));
        const float2 e = split2(pair_add(join2(exp2_approx(t.x), exp2_approx(t.y)), join2(low, low)));
        const Float2 s = pair_mul(join2(rcp_approx(e.x), rcp_approx(e.y)), join2(low, low));
        const Float2 a = pair_mul(g, s);
        if constexpr (GRAD) d = pair_fma(a, pair_fma(s, join2(-1.f, -1.f), join2(1.f, 1.f)), s);
        return a;
    } else if constexpr (ACT == GLU_GELU) {
        auto both = [](float c) { return join2(c, c); };
        const float2 v = split2(g);
        const float2 den = split2(pair_fma(join2(fabsf(v.x), fabsf(v.y)), both(0.23334524f), both(1.f)));
        const Float2 t = join2(rcp_approx(den.x), rcp_approx(den.y));
        const Float2 y = pair_mul(g, both(0.84932180f));  // e^(-g^2 / 2) = 2^(-y^2)
        const float2 y2 = split2(pair_mul(y, y));
        const Float2 e = join2(exp2_approx(-y2.x), exp2_approx(-y2.y));
        Float2 q = pair_fma(both(-0.06767226f), t, both(0.2301162f));
        q = pair_fma(q, t, both(-0.17557096f));
        q = pair_fma(q, t, both(0.20424654f));
        q = pair_fma(q, t, both(0.02361209f));
        q = pair_fma(q, t, both(0.10061143f));
        q = pair_fma(q, t, both(0.09147805f));
        q = pair_fma(q, t, both(0.0931789f));
        const float2 tail = split2(pair_mul(pair_mul(q, t), e));  // Phi(-|g|)
        const Float2 c = join2(v.x > 0.f ? 1.f - tail.x : tail.x, v.y > 0.f ? 1.f - tail.y : tail.y);
        if constexpr (GRAD) d = pair_fma(pair_mul(g, both(0.39894228f)), e, c);
        return pair_mul(g, c);
    } else {
        const float2 v = split2(g);
        float2 a, dd = make_float2(0.f, 0.f);
        auto one = [](float x, float& dx) {
            const float r = x > 0.f || x != x ? x : 0.f;  // NaN stays
            if constexpr (ACT == GLU_RELU) {
                if constexpr (GRAD) dx = x > 0.f ? 1.f : x != x ? x : 0.f;
                return r;
            } else {
                if constexpr (GRAD) dx = 2.f * r;
                return r * r;
            }
        };
        a.x = one(v.x, dd.x);
        a.y = one(v.y, dd.y);
        if constexpr (GRAD) d = join2(dd.x, dd.y);
        return join2(a.x, a.y);
    }
}
template <int ACT>
__device__ __forceinline__ float glu_act(float g) {
    Float2 unused;
    return split2(glu_act2<ACT, false>(join2(g, g), unused)).x;
}

}  // namespace sffn
