// AdamW over many tensors in one launch (gfx950): decoupled weight decay, moments in
// fp32 or in 8 bits, parameters in fp32 or in bf16 with an optional fp32 master.
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,
//   p = (1 - lr wd) p - (lr / c1) m / (sqrt(v) / sqrt(c2) + eps),  ck = 1 - bk^step.
//
// Moments in 8 bits: a block of 256 elements of a tensor shares A, its largest
// magnitude; a code c stands for A sign(c) (c / 127)^2 (m, int8) or A (c / 255)^4
// (v, uint8). The codes are thus equally spaced in the square (fourth) root: the
// step between neighbours is 1.6 % of a value at the top of the range and grows
// towards its low end, which reaches 6e-5 A (m) and 2e-10 A (v, whose square root
// divides). A second moment under 1.5e-11 A is held as 0: the gradient of the step, which
// enters in fp32, and eps then bound that element's update. A block of largest magnitude
// under 2^-120 is held as zeros; one with a NaN or an infinity becomes NaN as a whole.
//
// Rounded to the nearest code, a moment loses every change of less than half a code while A
// holds: at b2 = 0.999 a step takes 0.001 of v, a code is 4 / c of it, so v falls with A alone,
// and rises only where g^2 passes about 9 v (c = 255) to 40 v (c = 50); at b1 = 0.9 m stays
// where it is from |c| = 9 down. An element whose gradients grow from 0.1 to 0.4 of the block's
// largest then moves 3.6 times as far as it should, one whose gradients end keeps moving, for
// good. Unbiased rounding instead takes the upper of the two codes around a value
// with the probability of where the value is between theirs, so that the moments are right on average over
// steps. Its random words are a hash of the step, the tensor's place in the list and the
// element, so results repeat. A second moment that is not 0 is then never rounded to 0 (a
// first moment of one code over a second of none would be a step of any size): elements whose
// gradients are under 1.5e-5 of the block's largest move less than they should.
// Everything is computed in fp32 and rounds operation by operation in the order written
// (no fused products, IEEE quotients and roots), so that codes depend on the inputs alone.
//
// Bound by memory: each word is read once and written once. 50 M bf16 parameters with fp32
// masters and moments in 8 bits (18 bytes each, 0.91 GB) take 188 us, 4.8 TB/s where a copy
// reaches 5.2, and 225 with unbiased rounding, whose hashes and comparisons memory does not
// hide; 4.7 M in fp32 (28 bytes, 132 MB, held by the last cache) 21 us. A table of
// tensors in the kernel's arguments makes one launch of up to 48 tensors, so that small
// ones fill the device together and nothing is uploaded for the call.
#include "gs_host.h"

namespace gs {
namespace {

constexpr int kThreads = 256, kBlock = 256;  // kBlock: elements that share a scale, 4 to a lane of a wave
constexpr int kChunk = 2048;                 // elements of one workgroup
constexpr int64_t kMostGroups = 1 << 23;     // workgroups of one launch
constexpr int kTensors = 48;                 // tensors of one launch: their table fits the 4 KiB of kernel arguments

struct Table {
  gs_adamw_tensor t[kTensors];
  uint32_t first[kTensors];  // first workgroup of each tensor
  uint32_t key[kTensors];    // of its random words in this step
  int count;
};

enum { kWords = 0, kNearest = 1, kUnbiased = 2 };  // moments in fp32, or codes and their rounding

// A permutation of 32-bit words in which each bit of x changes each bit of the result half the
// time (over 20000 words to within 0.003): shifts and products with the fractions of the roots of 2 and 3.
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x = (x ^ x >> 16) * 0x6a09e667u;
  x = (x ^ x >> 15) * 0xbb67ae85u;
  return x ^ x >> 16;
}
constexpr uint32_t kGolden = 0x9e3779b9u;  // 2^32 over the golden ratio: spreads consecutive numbers
uint32_t key_of(int64_t step, int64_t tensor) {
  return mix(mix((uint32_t)step) + (uint32_t)tensor * kGolden + (uint32_t)(step >> 32));
}
// Element e's word for the first moment; that of the second is it times kGolden.
__device__ __forceinline__ uint32_t random_word(uint32_t key, int64_t e) {
  return mix(key + (uint32_t)e * kGolden + (uint32_t)(e >> 32));
}
__device__ __forceinline__ float uniform(uint32_t w) { return (float)(w >> 8) * 0x1p-24f; }  // [0, 1)

struct Scalars {
  float b1, c1m, b2, c2m, decay, root, eps, rate;  // b, 1 - b, 1 - lr wd, 1 / sqrt(c2), lr / c1
  const float* grad_scale;
};

typedef unsigned int u4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int u2u __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned int u1u __attribute__((aligned(1)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));

// Four elements at any alignment that the type allows; those past n read 0.
__device__ __forceinline__ void load4(const float* p, int64_t e, int64_t n, float (&x)[4]) {
  if (e + 4 <= n) {
    const u4u w = *reinterpret_cast<const u4u*>(p + e);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = e + i < n ? p[e + i] : 0.0f;
  }
}
__device__ __forceinline__ void load4(const __bf16* p, int64_t e, int64_t n, float (&x)[4]) {
  if (e + 4 <= n) {
    const u2u w = *reinterpret_cast<const u2u*>(p + e);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = e + i < n ? (float)p[e + i] : 0.0f;
  }
}
__device__ __forceinline__ uint32_t load4(const uint8_t* p, int64_t e, int64_t n) {
  if (e + 4 <= n) return *reinterpret_cast<const u1u*>(p + e);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= e + i < n ? (uint32_t)p[e + i] << (8 * i) : 0u;
  return w;
}
__device__ __forceinline__ void store4(float* p, int64_t e, int64_t n, const float (&x)[4]) {
  if (e + 4 <= n) {
    u4u w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(x[i]);
    *reinterpret_cast<u4u*>(p + e) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e + i < n) p[e + i] = x[i];
  }
}
__device__ __forceinline__ void store4(__bf16* p, int64_t e, int64_t n, const float (&x)[4]) {
  if (e + 4 <= n) {
    u2u w;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w[i] = __builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{x[2 * i], x[2 * i + 1]}), bf2v));
    *reinterpret_cast<u2u*>(p + e) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e + i < n) p[e + i] = (__bf16)x[i];
  }
}
__device__ __forceinline__ void store4(uint8_t* p, int64_t e, int64_t n, uint32_t w) {
  if (e + 4 <= n) {
    *reinterpret_cast<u1u*>(p + e) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (e + i < n) p[e + i] = (uint8_t)(w >> (8 * i));
  }
}

constexpr float kTiny = 0x1p-120f;
constexpr float kUnitM = (float)(1.0 / (127.0 * 127.0)), kUnitV = (float)(1.0 / (255.0 * 255.0 * 255.0 * 255.0));

template <bool QUARTIC>
__device__ __forceinline__ void values(uint32_t w, float scale, float (&x)[4]) {
#pragma clang fp contract(off)
  const float unit = scale * (QUARTIC ? kUnitV : kUnitM);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (QUARTIC) {
      const float c = (float)((w >> (8 * i)) & 255u), s = c * c;
      x[i] = s * s * unit;
    } else {
      const float c = (float)(int8_t)(w >> (8 * i));
      x[i] = c * __builtin_fabsf(c) * unit;
    }
  }
}

// Codes of a wave's 256 elements, four to a lane, and their block's scale. The largest
// magnitude is taken over bit patterns, in which infinity and NaN are above every number;
// with either the scale is NaN, and so is every value of the block. UNBIASED: `key` and e, the
// first of the lane's elements, give the random words.
template <bool QUARTIC, bool UNBIASED>
__device__ __forceinline__ uint32_t codes(const float (&x)[4], float* scale, uint32_t key, int64_t e) {
#pragma clang fp contract(off)
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) most = max(most, (uint32_t)__shfl_xor((int)most, d));
  const float A = most >= 0x7f800000u ? __builtin_nanf("") : __uint_as_float(most);
  const bool none = A < kTiny;
  const float inv = none ? 0.0f : 1.0f / A;
  *scale = none ? 0.0f : A;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float part = __builtin_fabsf(x[i]) * inv;
    float r = __builtin_sqrtf(part);
    if constexpr (QUARTIC) r = __builtin_sqrtf(r);
    constexpr float levels = QUARTIC ? 255.0f : 127.0f;
    int c;
    if constexpr (UNBIASED) {
      // between the values of codes lo and lo + 1, in units of code 1's
      const float lo = __builtin_fminf(__builtin_floorf(r * levels), levels - 1.0f), up = lo + 1.0f;
      const float l2 = lo * lo, u2 = up * up;
      const float below = QUARTIC ? l2 * l2 : l2, above = QUARTIC ? u2 * u2 : u2;
      const float at = part * (QUARTIC ? levels * levels * levels * levels : levels * levels);
      const uint32_t w = random_word(key, e + i);
      c = (int)lo + (uniform(QUARTIC ? w * kGolden : w) * (above - below) < at - below ? 1 : 0);
      if ((__float_as_uint(x[i]) & 0x7fffffffu) == most) c = (int)levels;
      if (QUARTIC && x[i] > 0.0f) c = max(c, 1);
      if (none) c = 0;
    } else {
      c = (int)__builtin_fminf(__builtin_rintf(r * levels), levels);
    }
    if (!QUARTIC && x[i] < 0.0f) c = -c;
    w |= ((uint32_t)c & 255u) << (8 * i);
  }
  return w;
}

// P: the parameter's type, G: the gradient's. MASTER: the parameter is the rounded copy
// of an fp32 master. Four elements a lane, so that a wave holds one block of 256.
template <typename P, typename G, bool MASTER, int CODES>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Table tab, Scalars s) {
#pragma clang fp contract(off)
  constexpr bool BYTES = CODES != kWords;
  int lo = 0, hi = tab.count - 1;  // the tensor whose workgroups hold this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first[mid] <= blockIdx.x)
      lo = mid;
    else
      hi = mid - 1;
  }
  const gs_adamw_tensor t = tab.t[lo];
  float gs = 1.0f;
  if (s.grad_scale != nullptr) {
    gs = *s.grad_scale;
    if (!(__builtin_fabsf(gs) < __builtin_inff())) return;  // uniform: the step is skipped
  }
  const int64_t n = t.n;
  const int64_t chunk = (int64_t)(blockIdx.x - tab.first[lo]) * kChunk;
#pragma unroll
  for (int u = 0; u < kChunk / (4 * kThreads); ++u) {
    const int64_t b = chunk + (int64_t)(u * kThreads + (threadIdx.x & ~63u)) * 4;  // the wave's block
    if (b >= n) return;  // uniform in the wave
    const int64_t e = b + 4 * (threadIdx.x & 63);
    float p[4], g[4], m[4], v[4];
    if constexpr (MASTER)
      load4(t.master, e, n, p);
    else
      load4(static_cast<const P*>(t.param), e, n, p);
    load4(static_cast<const G*>(t.grad), e, n, g);
    if constexpr (BYTES) {
      const int64_t q = b / kBlock;
      values<false>(load4(static_cast<const uint8_t*>(t.exp_avg), e, n), t.exp_avg_scale[q], m);
      values<true>(load4(static_cast<const uint8_t*>(t.exp_avg_sq), e, n), t.exp_avg_sq_scale[q], v);
    } else {
      load4(static_cast<const float*>(t.exp_avg), e, n, m);
      load4(static_cast<const float*>(t.exp_avg_sq), e, n, v);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float gi = s.grad_scale != nullptr ? g[i] * gs : g[i];
      m[i] = m[i] * s.b1 + gi * s.c1m;
      v[i] = v[i] * s.b2 + gi * gi * s.c2m;
      p[i] = p[i] * s.decay - m[i] / (__builtin_sqrtf(v[i]) * s.root + s.eps) * s.rate;
    }
    if constexpr (MASTER) store4(t.master, e, n, p);
    store4(static_cast<P*>(t.param), e, n, p);
    if constexpr (BYTES) {
      const int64_t q = b / kBlock;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e + i >= n) m[i] = v[i] = 0.0f;
      float sm, sv;
      const uint32_t cm = codes<false, CODES == kUnbiased>(m, &sm, tab.key[lo], e);
      const uint32_t cv = codes<true, CODES == kUnbiased>(v, &sv, tab.key[lo], e);
      store4(static_cast<uint8_t*>(t.exp_avg), e, n, cm);
      store4(static_cast<uint8_t*>(t.exp_avg_sq), e, n, cv);
      if ((threadIdx.x & 63) == 0) {
        t.exp_avg_scale[q] = sm;
        t.exp_avg_sq_scale[q] = sv;
      }
    } else {
      store4(static_cast<float*>(t.exp_avg), e, n, m);
      store4(static_cast<float*>(t.exp_avg_sq), e, n, v);
    }
  }
}

template <bool QUARTIC>
__global__ __launch_bounds__(kThreads) void adamw_values_kernel(const uint8_t* codes_, const float* scale, float* out,
                                                                int64_t n) {
  const int64_t e = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4;
  if (e >= n) return;
  float x[4];
  values<QUARTIC>(load4(codes_, e, n), scale[e / kBlock], x);
  store4(out, e, n, x);
}

typedef void (*AdamwFn)(Table, Scalars);

AdamwFn kernel_of(int pd, int gd, bool master, int codes) {
#define GS_ADAMW(P, G, M) (codes == kUnbiased ? adamw_kernel<P, G, M, kUnbiased> : codes == kNearest ? adamw_kernel<P, G, M, kNearest> : adamw_kernel<P, G, M, kWords>)
  const bool gf = gd == GS_DTYPE_F32;
  if (pd == GS_DTYPE_F32) return gf ? GS_ADAMW(float, float, false) : GS_ADAMW(float, __bf16, false);
  if (master) return gf ? GS_ADAMW(__bf16, float, true) : GS_ADAMW(__bf16, __bf16, true);
  return gf ? GS_ADAMW(__bf16, float, false) : GS_ADAMW(__bf16, __bf16, false);
#undef GS_ADAMW
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_adamw_step(const gs_adamw_args* a, hipStream_t stream) {
  const char* who = "gs_adamw_step";
  clear_error();
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  if (a->count < 0 || (a->count > 0 && a->tensors == nullptr))
    return set_error(GS_ERR_INVALID, "%s: tensors must be an array of count >= 0", who);
  if ((a->param_dtype != GS_DTYPE_F32 && a->param_dtype != GS_DTYPE_BF16) ||
      (a->grad_dtype != GS_DTYPE_F32 && a->grad_dtype != GS_DTYPE_BF16))
    return set_error(GS_ERR_INVALID, "%s: unknown dtype (%d, %d)", who, a->param_dtype, a->grad_dtype);
  if (a->state_bits != 8 && a->state_bits != 32)
    return set_error(GS_ERR_INVALID, "%s: state_bits must be 8 or 32; got %d", who, a->state_bits);
  if (a->has_master && a->param_dtype != GS_DTYPE_BF16)
    return set_error(GS_ERR_INVALID, "%s: masters belong to bfloat16 parameters", who);
  if (a->step < 1) return set_error(GS_ERR_INVALID, "%s: step counts from 1; got %lld", who, (long long)a->step);
  if (!(a->beta1 >= 0.0 && a->beta1 < 1.0) || !(a->beta2 >= 0.0 && a->beta2 < 1.0))
    return set_error(GS_ERR_INVALID, "%s: betas must be in [0, 1); got (%g, %g)", who, a->beta1, a->beta2);
  if (!(a->lr >= 0.0 && std::isfinite(a->lr)) || !(a->eps >= 0.0 && std::isfinite(a->eps)) ||
      !(a->weight_decay >= 0.0 && std::isfinite(a->weight_decay)))
    return set_error(GS_ERR_INVALID, "%s: lr, eps and weight_decay must be finite and >= 0; got %g, %g, %g", who, a->lr,
                     a->eps, a->weight_decay);
  if (a->rounding != GS_ROUND_NEAREST && a->rounding != GS_ROUND_UNBIASED)
    return set_error(GS_ERR_INVALID, "%s: unknown rounding %d", who, a->rounding);
  const bool bytes = a->state_bits == 8;
  for (int64_t i = 0; i < a->count; ++i) {
    const gs_adamw_tensor& t = a->tensors[i];
    if (t.n < 0 || t.n > kMostGroups * kChunk)
      return set_error(GS_ERR_INVALID, "%s: tensor %lld has %lld elements", who, (long long)i, (long long)t.n);
    if (t.n > 0 && (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || (bytes && (!t.exp_avg_scale || !t.exp_avg_sq_scale)) ||
                    (a->has_master && !t.master)))
      return set_error(GS_ERR_INVALID, "%s: tensor %lld has a NULL pointer", who, (long long)i);
  }
  const double c1 = 1.0 - std::pow(a->beta1, (double)a->step), c2 = 1.0 - std::pow(a->beta2, (double)a->step);
  Scalars s;
  s.b1 = (float)a->beta1;
  s.c1m = (float)(1.0 - a->beta1);
  s.b2 = (float)a->beta2;
  s.c2m = (float)(1.0 - a->beta2);
  s.decay = (float)(1.0 - a->lr * a->weight_decay);
  s.root = (float)std::pow(c2, -0.5);
  s.eps = (float)a->eps;
  s.rate = (float)(a->lr / c1);
  s.grad_scale = a->grad_scale;
  const AdamwFn fn = kernel_of(a->param_dtype, a->grad_dtype, a->has_master != 0,
                               !bytes ? kWords : a->rounding == GS_ROUND_UNBIASED ? kUnbiased : kNearest);
  Table tab;
  tab.count = 0;
  int64_t groups = 0;
  auto flush = [&]() -> int {
    if (groups == 0) return GS_OK;
    hipLaunchKernelGGL(fn, dim3((unsigned)groups), dim3(kThreads), 0, stream, tab, s);
    GS_CHECK_HIP(hipGetLastError());
    tab.count = 0;
    groups = 0;
    return GS_OK;
  };
  for (int64_t i = 0; i < a->count; ++i) {
    const gs_adamw_tensor& t = a->tensors[i];
    if (t.n == 0) continue;
    const int64_t need = (t.n + kChunk - 1) / kChunk;
    if (tab.count == kTensors || groups + need > kMostGroups) {
      const int rc = flush();
      if (rc) return rc;
    }
    tab.t[tab.count] = t;
    tab.key[tab.count] = key_of(a->step, i);
    tab.first[tab.count++] = (uint32_t)groups;
    groups += need;
  }
  return flush();
}

extern "C" int gs_adamw_dequantize(const void* codes, const float* scale, float* out, int64_t n, int32_t second,
                                   hipStream_t stream) {
  const char* who = "gs_adamw_dequantize";
  clear_error();
  if (n < 0 || n > kMostGroups * 4 * kThreads)
    return set_error(GS_ERR_INVALID, "%s: bad count %lld", who, (long long)n);
  if (n == 0) return GS_OK;
  if (!codes || !scale || !out)
    return set_error(GS_ERR_INVALID, "%s: codes, scale and out must be non-NULL device pointers", who);
  auto fn = second ? adamw_values_kernel<true> : adamw_values_kernel<false>;
  hipLaunchKernelGGL(fn, dim3((unsigned)((n + 4 * kThreads - 1) / (4 * kThreads))), dim3(kThreads), 0, stream,
                     static_cast<const uint8_t*>(codes), scale, out, n);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}
