// Building blocks of the operators over sequences of tokens (convolution, selective scan,
// embedding, token log probabilities): typed loads and stores that end at a row's end, sums
// over the lanes of a wave, softplus, and checks of strides.
#pragma once

#include "gs_host.h"

namespace gs {

// One element of type T in a buffer access, held as a word until it is needed so that many
// loads can be in flight. An offset of kOffNone reads 0 and writes nothing.
template <typename T>
struct Elem {
  static __device__ __forceinline__ unsigned int load(const void* base, uint32_t off) {
    const auto r = bounded_rsrc(base, 0x7fffffffu);
    if constexpr (sizeof(T) == 2)
      return (unsigned int)(unsigned short)__builtin_amdgcn_raw_buffer_load_b16(r, (int)off, 0, 0);
    else
      return __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0);
  }
  static __device__ __forceinline__ void store(void* base, uint32_t off, float x) {
    const auto r = bounded_rsrc(base, 0x7fffffffu);
    if constexpr (sizeof(T) == 2)
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (__bf16)x), r, (int)off, 0, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), r, (int)off, 0, 0);
  }
  static __device__ __forceinline__ float value(unsigned int w) { return __uint_as_float(sizeof(T) == 2 ? w << 16 : w); }
};

// A workgroup barrier that orders LDS alone (global loads stay in flight), for the compiler too:
// values read from LDS before it are read again after it.
__device__ __forceinline__ void share_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The same between the lanes of one wave, whose LDS accesses keep their order by themselves: for the compiler
// alone, no instruction.
__device__ __forceinline__ void share_in_wave() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// In lanes whose bit M is clear a[l] + a[l ^ M], in the others b[l] + b[l ^ M]: six of these,
// each over half as many registers as the one before, leave 64 sums over a wave in one register.
template <int M>
__device__ __forceinline__ float join(float a, float b) {
  if constexpr (M >= 16) {
    typedef unsigned int u2 __attribute__((ext_vector_type(2)));
    const u2 s = M == 32 ? __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false)
                         : __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
  } else {
    const bool up = (__lane_id() & M) != 0;
    return (up ? b : a) + lane_xor_c<M>(up ? a : b);
  }
}

// log(1 + e^x) = max(x, 0) + log(1 + e) with e = e^-|x|, and log(1 + e) = 2 artanh(s) with
// s = e / (2 + e) <= 1/3 by its series (the first term left out is 2e-9 of the sum): a step size of
// 1e-4 keeps all its digits, which the logarithm of a rounded 1 + e would lose.
__device__ __forceinline__ float softplus(float x) {
  const float e = __builtin_amdgcn_exp2f(-kLog2e * __builtin_fabsf(x));
  const float s = e * __builtin_amdgcn_rcpf(2.0f + e), t = s * s;
  float p = __builtin_fmaf(t, 1.0f / 15, 1.0f / 13);
  p = __builtin_fmaf(p, t, 1.0f / 11);
  p = __builtin_fmaf(p, t, 1.0f / 9);
  p = __builtin_fmaf(p, t, 1.0f / 7);
  p = __builtin_fmaf(p, t, 1.0f / 5);
  p = __builtin_fmaf(p, t, 1.0f / 3);
  p = __builtin_fmaf(p, t, 1.0f);
  return __builtin_fmaf(2.0f * s, p, x < 0.0f ? 0.0f : x);  // a NaN passes
}

// Rows of `n` elements at t * st + b * sb: written ones must not overlap each other.
inline int check_step_rows(const char* who, const char* name, int64_t T, int64_t B, int64_t n, int64_t st, int64_t sb,
                           bool written) {
  if (st < 0 || sb < 0)
    return set_error(GS_ERR_INVALID, "%s: %s has a negative stride (%lld, %lld)", who, name, (long long)st, (long long)sb);
  if (written && ((B > 1 && T > 1 && !(st >= sb * (B - 1) + n && sb >= n) && !(sb >= st * (T - 1) + n && st >= n)) ||
                  (B > 1 && sb < n) || (T > 1 && st < n)))
    return set_error(GS_ERR_INVALID, "%s: %s rows overlap (strides %lld, %lld)", who, name, (long long)st, (long long)sb);
  return GS_OK;
}

inline int check_dtype(const char* who, int dtype) {
  if (dtype != GS_DTYPE_F32 && dtype != GS_DTYPE_BF16)
    return set_error(GS_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
  return GS_OK;
}

inline int check_plain_scratch(const char* who, const void* scratch, int64_t have, int64_t need) {
  if (need > 0 && (scratch == nullptr || have < need || (reinterpret_cast<uintptr_t>(scratch) & 255u) != 0))
    return set_error(GS_ERR_INVALID, "%s: scratch of %lld bytes, 256-byte aligned, required; got %lld at %p", who,
                     (long long)need, (long long)have, scratch);
  return GS_OK;
}

}  // namespace gs
