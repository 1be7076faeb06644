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
  int M = 0, N = 0, K = 0, ksplit = 1, layout = kGemmNT;
};

// Splits of K with which a product fills the device (1: none).
int gemm_bf16_pick_split(int M, int N, int K);
int gemm_bf16(const GemmBf16Args& g, hipStream_t stream, const char* who);

// The activations, and their derivatives at the same argument.
__device__ __forceinline__ float act_value(float x, int act) {
  switch (act) {
    case GS_ACT_TANH: return tanh_near(x);
    case GS_ACT_RELU: return x < 0.0f ? 0.0f : x;  // a NaN passes
    case GS_ACT_GELU: return 0.5f * x * (1.0f + erff(x * 0.70710678f));
    case GS_ACT_SILU: return x * sigmoid(x);
    case GS_ACT_SIGMOID: return sigmoid(x);
    default: return x;
  }
}
__device__ __forceinline__ float act_slope(float x, int act) {
  switch (act) {
    case GS_ACT_TANH: {
      const float y = tanh_near(x);
      return __builtin_fmaf(-y, y, 1.0f);
    }
    case GS_ACT_RELU: return x > 0.0f ? 1.0f : 0.0f;
    case GS_ACT_GELU: {
      const float phi = 0.39894228f * __builtin_amdgcn_exp2f(x * x * (-0.5f * kLog2e));
      return __builtin_fmaf(x, phi, 0.5f * (1.0f + erff(x * 0.70710678f)));
    }
    case GS_ACT_SILU: {
      const float s = sigmoid(x);
      return s * __builtin_fmaf(x, 1.0f - s, 1.0f);
    }
    case GS_ACT_SIGMOID: {
      const float s = sigmoid(x);
      return s * (1.0f - s);
    }
    default: return 1.0f;
  }
}

}  // namespace gs
