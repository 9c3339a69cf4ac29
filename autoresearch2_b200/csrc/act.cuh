// The gated feed-forward block's activations and their derivatives, float32.
#pragma once

#include "common.cuh"

namespace sffn {

enum { GLU_RELU = 0, GLU_RELU2 = 1, GLU_SILU = 2, GLU_GELU = 3 };

// act(g) and act'(g).  SiLU: s = 1 / (1 + exp(-g)), the hardware's exp2 and
// reciprocal (a few 2^-22 of the value: below a twentieth of a 16-bit
// rounding).  GELU is the exact one; erfc keeps its relative precision where
// 1 + erf would cancel.
template <int ACT, bool GRAD>
__device__ __forceinline__ float glu_act(float g, float& d) {
    if constexpr (ACT == GLU_SILU) {
        const float s = __fdividef(1.f, 1.f + __expf(-g));
        const float a = g * s;
        if constexpr (GRAD) d = fmaf(a, 1.f - s, s);
        return a;
    } else if constexpr (ACT == GLU_GELU) {
        const float c = 0.5f * erfcf(-0.70710678118654752f * g);
        if constexpr (GRAD) d = fmaf(g * 0.39894228040143268f, __expf(-0.5f * g * g), c);
        return g * c;
    } else {
        const float r = g > 0.f || g != g ? g : 0.f;  // NaN stays
        if constexpr (ACT == GLU_RELU) {
            if constexpr (GRAD) d = g > 0.f ? 1.f : g != g ? g : 0.f;
            return r;
        } else {
            if constexpr (GRAD) d = 2.f * r;
            return r * r;
        }
    }
}

}  // namespace sffn
