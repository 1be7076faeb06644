// bf16 products with fp32 sums for the linear operator (gemm_bf16.hip):
//   C[i, j] = sum_k A(i, k) B(k, j)
// in the layouts of GemmLayout (gs_gemm.h), followed by
//   pre = C + bias[j] (stored to `pre` where asked), y = act(pre) + residual[i, j].
#pragma once

#include "gs_gemm.h"

namespace gs {

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
// NT products of so few rows of A are read from memory straight into the matrix units: no
// splits, no copies.
bool gemm_bf16_few_rows(int M, int N, int K);
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

// pre of a bf16 call, kept for its backward in 16 bits: a half, three bits more than a bf16 has,
// which is what act' needs of it (in bf16 the gradients' error against 64 bits, 0.00235 from
// rounding dpre and the gradients themselves, is 0.0024 with silu and 0.0026 with tanh). Beyond a
// half's range act' is constant: larger values are held as its largest, smaller ones, but 0, as
// its smallest, whose sign relu needs.
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned int kept_pair(float a, float b) {
  typedef float f2v __attribute__((ext_vector_type(2)));
  auto fit = [](float x) __attribute__((always_inline)) {
    const float in = __builtin_copysignf(__builtin_fminf(__builtin_fmaxf(__builtin_fabsf(x), 0x1p-24f), 65504.0f), x);
    return x != x || x == 0.0f ? x : in;
  };
  return __builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{fit(a), fit(b)}), half2v));
}
__device__ __forceinline__ void kept_floats(const Granule& w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned int word = w[i];  // a bit cast of w[i] itself takes w[0]'s bits
    const half2v h = __builtin_bit_cast(half2v, word);
    x[2 * i] = (float)h[0];
    x[2 * i + 1] = (float)h[1];
  }
}

// dx (NN) and dw (TN) of a backward whose tiles are all small, and the column sums, in one
// launch (and the splits' sum of dw): M = 2048, N = 1024, K = 512 takes 12.6 + 9.3 + 3.9
// us in three.
bool gemm_bf16_pair_applies(const GemmBf16Args& x, const GemmBf16Args& w);
int gemm_bf16_pair(const GemmBf16Args& x, const GemmBf16Args& w, const ColumnSums& c, hipStream_t stream, const char* who);

}  // namespace gs
