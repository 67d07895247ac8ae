// act.cuh -- the activations that the fused layers apply (J4C_ACT_*), and
// their derivatives.  FLOAT32 tanh and sigmoid are the elementwise kernels'
// (jmath.cuh; their error bounds are there); FLOAT64 uses CUDA's tanh and exp.
//
//   silu(u) = u sigmoid(u);  gelu(u) = u sigmoid(2 a(u)), a(u) = sqrt(2/pi) (u + 0.044715 u^3), which is the tanh
//   form u/2 (1 + tanh a(u)) without its cancellation for negative u.
//   With s the sigmoid: silu' = s + u s (1 - s), gelu' = s + u s (1 - s) 2 a'(u).
#pragma once

#include "common.cuh"
#include "jmath.cuh"

namespace j4c {

J4C_MATH_DEFS

__device__ __forceinline__ float act_tanh(float x) { return j_tanh(x); }
__device__ __forceinline__ double act_tanh(double x) { return tanh(x); }
__device__ __forceinline__ float act_sigmoid(float x) { return j_sigmoid(x); }
__device__ __forceinline__ double act_sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }

// 2 a(u) and 2 a'(u)
template <typename T>
__device__ __forceinline__ T gelu_arg(T u) {
    return T(1.5957691216057308) * (u + T(0.044715) * u * u * u);
}
template <typename T>
__device__ __forceinline__ T gelu_arg_slope(T u) {
    return T(1.5957691216057308) * (T(1) + T(0.134145) * u * u);
}

template <typename T>
__device__ __forceinline__ T act_value(int act, T u) {
    switch (act) {
    case J4C_ACT_RELU: return T(0) >= u ? T(0) : u;  // NaN stays
    case J4C_ACT_TANH: return act_tanh(u);
    case J4C_ACT_SIGMOID: return act_sigmoid(u);
    case J4C_ACT_SILU: return u * act_sigmoid(u);
    case J4C_ACT_GELU: return u * act_sigmoid(gelu_arg(u));
    default: return u;
    }
}

// The derivative at the pre-activation u.
template <typename T>
__device__ __forceinline__ T act_slope(int act, T u) {
    switch (act) {
    case J4C_ACT_RELU: return u > T(0) ? T(1) : T(0);
    case J4C_ACT_TANH: {
        const T t = act_tanh(u);
        return T(1) - t * t;
    }
    case J4C_ACT_SIGMOID: {
        const T s = act_sigmoid(u);
        return s * (T(1) - s);
    }
    case J4C_ACT_SILU: {
        const T s = act_sigmoid(u);
        return s + u * (s * (T(1) - s));
    }
    case J4C_ACT_GELU: {
        const T s = act_sigmoid(gelu_arg(u)), q = s * (T(1) - s);
        return q == T(0) ? s : s + u * q * gelu_arg_slope(u);  // q = 0: far out, where a' may overflow
    }
    default: return T(1);
    }
}

inline bool act_known(int act) { return act >= J4C_ACT_NONE && act <= J4C_ACT_GELU; }

}  // namespace j4c
