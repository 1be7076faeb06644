// bf16 products with fp32 sums for the linear operator (gemm_bf16.hip):
//   C[i, j] = sum_k A(i, k) B(k, j)
// in the layouts of GemmLayout (gs_gemm.h), followed by
//   pre = C + bias[j] (stored to `pre` where asked), y = act(pre) + residual[i, j].
#pragma once

#include "gs_gemm.h"

namespace gs {

struct LinearEpilogue {
  const void* bias = nullptr;      // [N]
  const void* residual = nullptr;  // [M, N], row stride ldr
  void* pre = nullptr;             // [M, N] contiguous
  int64_t ldr = 0;
  int act = GS_ACT_NONE;
};

struct GemmBf16Args {
  const __bf16* a = nullptr;
  int64_t lda = 0;
  const __bf16* b = nullptr;
  int64_t ldb = 0;
  __bf16* y = nullptr;  // ksplit == 1: [M, N], row stride ldy
  int64_t ldy = 0;
  float* part = nullptr;  // ksplit > 1: split s writes its sums to part + s M N ([M, N] contiguous)
  LinearEpilogue epi;
  bool a_pads = false, b_pads = false;  // zeros follow the operand's rows up to a multiple of 8 elements
  int M = 0, N = 0, K = 0, ksplit = 1, layout = kGemmNT;
};

// Splits of K with which a product fills the device (1: none).
int gemm_bf16_pick_split(int M, int N, int K);
int gemm_bf16(const GemmBf16Args& g, hipStream_t stream, const char* who);

// Granules: eight consecutive bf16 of a row, at any alignment. Where a row ends inside
// one, the row's last eight elements are loaded instead and moved down, zeros behind
// them: one load like any other (element by element, a tile at the edge of an operand
// took eight dependent loads a slice).
typedef unsigned int Granule __attribute__((ext_vector_type(4)));
typedef unsigned int GranuleAt __attribute__((ext_vector_type(4), aligned(2)));

// The load of the granule at p, `have` elements of which are in the row (any number; none:
// zeros) and `before` elements of the row in front of it; settle() with the same `have`
// then gives the granule.
__device__ __forceinline__ Granule granule_load(const __bf16* p, int have, int before) {
  Granule w = {0u, 0u, 0u, 0u};
  if (have >= 8) {
    w = *reinterpret_cast<const GranuleAt*>(p);
  } else if (have > 0) {
    if (before >= 8 - have) {
      w = *reinterpret_cast<const GranuleAt*>(p + have - 8);
    } else {  // a row of fewer than eight: its elements where settle() looks for them
      const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = i - (8 - have);
        if (at >= 0) w[i >> 1] |= (unsigned int)h[at] << (16 * (i & 1));
      }
    }
  }
  return w;
}
__device__ __forceinline__ Granule granule_settle(Granule w, int have) {
  const int down = have > 0 && have < 8 ? 8 - have : 0;
  if (down & 4) w = Granule{w[2], w[3], 0u, 0u};
  if (down & 2) w = Granule{w[1], w[2], w[3], 0u};
  if (down & 1) w = Granule{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16};
  return w;
}
__device__ __forceinline__ void granule_floats(const Granule& w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

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

}  // namespace gs
