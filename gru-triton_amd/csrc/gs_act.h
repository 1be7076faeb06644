// The linear operator's activations, their derivatives, what follows a product's sums, and
// sums over columns.
#pragma once

#include "gs_host.h"

namespace gs {

// pre = sums + bias[j] (stored to `pre` where asked), y = act(pre) + residual[i, j]. All but
// `pre` in the operands' type.
struct LinearEpilogue {
  const void* bias = nullptr;      // [N]
  const void* residual = nullptr;  // [M, N], row stride ldr
  void* pre = nullptr;             // [M, N] contiguous, halves where the type is bf16
  int64_t ldr = 0;
  int act = GS_ACT_NONE;
};

// The normal distribution's Phi(x) and phi(x) = Phi'(x), Phi within 8e-8: the rational
// approximation of erf in Abramowitz and Stegun, Handbook of Mathematical Functions,
// 7.1.26, at x / sqrt 2, whose exponential is that of phi.
__device__ __forceinline__ void normal(float x, float& Phi, float& phi) {
  const float a = __builtin_fabsf(x), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f * 0.70710678f, a, 1.0f));
  const float e = __builtin_amdgcn_exp2f(x * x * (-0.5f * kLog2e));
  float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
  p = __builtin_fmaf(p, t, 1.421413741f);
  p = __builtin_fmaf(p, t, -0.284496736f);
  p = __builtin_fmaf(p, t, 0.254829592f);
  const float q = 0.5f * p * t * e;  // 1 - Phi(|x|)
  Phi = x < 0.0f ? q : 1.0f - q;
  phi = 0.39894228f * e;
}

// The activations, and their derivatives at the same argument.
template <int ACT>
__device__ __forceinline__ float act_value(float x) {
  if constexpr (ACT == GS_ACT_TANH) return tanh_near(x);
  if constexpr (ACT == GS_ACT_RELU) return x < 0.0f ? 0.0f : x;  // a NaN passes
  if constexpr (ACT == GS_ACT_GELU) {
    float Phi, phi;
    normal(x, Phi, phi);
    return x * Phi;
  }
  if constexpr (ACT == GS_ACT_SILU) return x * sigmoid(x);
  if constexpr (ACT == GS_ACT_SIGMOID) return sigmoid(x);
  return x;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float x) {
  if constexpr (ACT == GS_ACT_TANH) {
    const float y = tanh_near(x);
    return __builtin_fmaf(-y, y, 1.0f);
  }
  if constexpr (ACT == GS_ACT_RELU) return x > 0.0f ? 1.0f : 0.0f;
  if constexpr (ACT == GS_ACT_GELU) {
    float Phi, phi;
    normal(x, Phi, phi);
    return __builtin_fmaf(x, phi, Phi);
  }
  if constexpr (ACT == GS_ACT_SILU) {
    const float s = sigmoid(x);
    return s * __builtin_fmaf(x, 1.0f - s, 1.0f);
  }
  if constexpr (ACT == GS_ACT_SIGMOID) {
    const float s = sigmoid(x);
    return s * (1.0f - s);
  }
  return 1.0f;
}

// f(std::integral_constant<int, act>) for the act of a launch (uniform).
template <typename F>
__device__ __forceinline__ void with_act(int act, F&& f) {
  switch (act) {
    case GS_ACT_TANH: f(std::integral_constant<int, GS_ACT_TANH>{}); break;
    case GS_ACT_RELU: f(std::integral_constant<int, GS_ACT_RELU>{}); break;
    case GS_ACT_GELU: f(std::integral_constant<int, GS_ACT_GELU>{}); break;
    case GS_ACT_SILU: f(std::integral_constant<int, GS_ACT_SILU>{}); break;
    case GS_ACT_SIGMOID: f(std::integral_constant<int, GS_ACT_SIGMOID>{}); break;
    default: f(std::integral_constant<int, GS_ACT_NONE>{});
  }
}
template <int N>
__device__ __forceinline__ void act_values(float (&x)[N], int act) {
  with_act(act, [&](auto A) __attribute__((always_inline)) {
#pragma unroll
    for (int v = 0; v < N; ++v) x[v] = act_value<decltype(A)::value>(x[v]);
  });
}
template <int N>
__device__ __forceinline__ void act_slopes(float (&x)[N], int act) {
  with_act(act, [&](auto A) __attribute__((always_inline)) {
#pragma unroll
    for (int v = 0; v < N; ++v) x[v] = act_slope<decltype(A)::value>(x[v]);
  });
}

// dst[e] = sum over parts of src[part * n + e], rounded to the tensor's type.
struct ColumnSums {
  void* dst = nullptr;
  const float* src = nullptr;
  int n = 0, parts = 0;
};

// Workgroup `group` of 256 threads takes 16 columns, its 16 part lanes every 16th part,
// joined through LDS in order.
template <typename T>
__device__ __forceinline__ void sum_columns(const ColumnSums& p, int group, float (*red)[17]) {
  const int c = threadIdx.x & 15, l = threadIdx.x >> 4, e = group * 16 + c;
  float s = 0.0f;
  if (e < p.n) {
    for (int k0 = l; k0 < p.parts; k0 += 16 * 8) {  // eight loads in flight
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = k0 + 16 * u < p.parts ? p.src[(int64_t)(k0 + 16 * u) * p.n + e] : 0.0f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += x[u];
    }
  }
  red[l][c] = s;
  __syncthreads();
  if (l == 0 && e < p.n) {
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][c];
    static_cast<T*>(p.dst)[e] = (T)s;
  }
}

}  // namespace gs
