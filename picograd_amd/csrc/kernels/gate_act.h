// The gate activations of the gated layer and their derivatives (device
// code): PGK_ACT_* plus SiLU and sigmoid, on pgmath.h's functions.
#ifndef PGK_GATE_ACT_H
#define PGK_GATE_ACT_H

#include <type_traits>

#include "launch.h"
#include "pgmath.h"

template <int ACT>
__device__ __forceinline__ float gate_f(float g)
{
    if constexpr (ACT == PGK_ACT_RELU)
        return g > 0.0f ? g : 0.0f;
    else if constexpr (ACT == PGK_ACT_GELU)
        return pgm_gelu(g);
    else if constexpr (ACT == PGK_ACT_SILU)
        return g * pgm_sigmoid(g);
    else if constexpr (ACT == PGK_ACT_SIGMOID)
        return pgm_sigmoid(g);
    else
        return g;
}

// act(g) and, in d, act'(g)
template <int ACT>
__device__ __forceinline__ float gate_fd(float g, float &d)
{
    if constexpr (ACT == PGK_ACT_RELU) {
        d = g > 0.0f ? 1.0f : 0.0f;
        return g > 0.0f ? g : 0.0f;
    } else if constexpr (ACT == PGK_ACT_GELU) {
        float density;
        const float cdf = pgm_Phi(g, &density);
        d = cdf + g * density;
        return g * cdf;
    } else if constexpr (ACT == PGK_ACT_SILU) {
        const float s = pgm_sigmoid(g);
        d = s * (1.0f + g * (1.0f - s));
        return g * s;
    } else if constexpr (ACT == PGK_ACT_SIGMOID) {
        const float s = pgm_sigmoid(g);
        d = s * (1.0f - s);
        return s;
    } else {
        d = 1.0f;
        return g;
    }
}

// the code as a template argument: fn(std::integral_constant<int, ACT>{})
template <class FN>
__device__ __forceinline__ void gate_switch(int act, FN fn)
{
    switch (act) {
    case PGK_ACT_RELU: fn(std::integral_constant<int, PGK_ACT_RELU>{}); break;
    case PGK_ACT_GELU: fn(std::integral_constant<int, PGK_ACT_GELU>{}); break;
    case PGK_ACT_SILU: fn(std::integral_constant<int, PGK_ACT_SILU>{}); break;
    case PGK_ACT_SIGMOID: fn(std::integral_constant<int, PGK_ACT_SIGMOID>{}); break;
    default: fn(std::integral_constant<int, PGK_ACT_NONE>{}); break;
    }
}

#endif
