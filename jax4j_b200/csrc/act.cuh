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

// u[i] <- act(u[i]) for N values: one branch on the activation for all of them.
template <typename T, int N>
__device__ __forceinline__ void act_values(int act, T (&u)[N]) {
    switch (act) {
    case J4C_ACT_RELU:
#pragma unroll
        for (int i = 0; i < N; i++) u[i] = T(0) >= u[i] ? T(0) : u[i];  // NaN stays
        break;
    case J4C_ACT_TANH:
#pragma unroll
        for (int i = 0; i < N; i++) u[i] = act_tanh(u[i]);
        break;
    case J4C_ACT_SIGMOID:
#pragma unroll
        for (int i = 0; i < N; i++) u[i] = act_sigmoid(u[i]);
        break;
    case J4C_ACT_SILU:
#pragma unroll
        for (int i = 0; i < N; i++) u[i] = u[i] * act_sigmoid(u[i]);
        break;
    case J4C_ACT_GELU:
#pragma unroll
        for (int i = 0; i < N; i++) u[i] = u[i] * act_sigmoid(gelu_arg(u[i]));
        break;
    default: break;
    }
}

// d[i] <- d[i] act'(u[i]), the derivative at the pre-activation u[i].
template <typename T, int N>
__device__ __forceinline__ void act_slopes(int act, const T (&u)[N], T (&d)[N]) {
    switch (act) {
    case J4C_ACT_RELU:
#pragma unroll
        for (int i = 0; i < N; i++) d[i] = u[i] > T(0) ? d[i] : T(0);  // Grad.reluGrad (api/Grad.java:593-597)
        break;
    case J4C_ACT_TANH:
#pragma unroll
        for (int i = 0; i < N; i++) {
            const T t = act_tanh(u[i]);
            d[i] *= T(1) - t * t;
        }
        break;
    case J4C_ACT_SIGMOID:
#pragma unroll
        for (int i = 0; i < N; i++) {
            const T s = act_sigmoid(u[i]);
            d[i] *= s * (T(1) - s);
        }
        break;
    case J4C_ACT_SILU:
#pragma unroll
        for (int i = 0; i < N; i++) {
            const T s = act_sigmoid(u[i]);
            d[i] *= s + u[i] * (s * (T(1) - s));
        }
        break;
    case J4C_ACT_GELU:
#pragma unroll
        for (int i = 0; i < N; i++) {
            const T s = act_sigmoid(gelu_arg(u[i])), q = s * (T(1) - s);
            d[i] *= q == T(0) ? s : s + u[i] * q * gelu_arg_slope(u[i]);  // q = 0: far out, where a' may overflow
        }
        break;
    default: break;
    }
}

inline bool act_known(int act) { return act >= J4C_ACT_NONE && act <= J4C_ACT_GELU; }

}  // namespace j4c
