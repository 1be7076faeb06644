// Log probabilities of given tokens (gfx950), from logits x [M, V]:
//   lse = log sum_v exp x_v,  logprob = x[token] - lse,  entropy = -sum_v p_v log p_v, p = exp(x - lse),
// with the `top` likeliest tokens of each row and theirs (of equal ones the lowest index first), and the gradient
//   dx_v = dlogprob ([v = token] - p_v) - dentropy p_v (log p_v + entropy).
// With d = x - max, s = sum exp d and t = sum d exp d: lse = max + log s, entropy = log s - t / s.
// A logit of -infinity is a token that cannot come: it adds nothing. A row of those alone has log
// probabilities -infinity, entropy 0 and no gradient. A NaN or +infinity makes a row NaN. A
// negative token marks a row whose token does not count: its log probability is 0, and sends no gradient. A row to which
// no gradient comes has none, also where its logits are NaN.
//
// Bound by memory: one pass over the logits forward with the running maximum, s and t, and one backward.
// A workgroup takes a row, or a part of one where there are few rows; the parts of a row are
// then joined in order. For `top` a part's logits stay in registers as sortable words; each wave takes
// the largest out of its 512 or 2048 one after the other, and lists are merged, of waves and then of parts.
// 8192 rows of 32000 bf16: forward 126 to 145 us (3.6 to 4.2 TB/s of reads; a read alone reached 4.0), backward 189 (5.5 TB/s);
// 8 rows with the 8 likeliest 9 + 6, where launches and the chains of comparisons count.
#include "gs_seq.h"

namespace gs {
namespace {

typedef unsigned int u4v __attribute__((ext_vector_type(4)));

constexpr int kMostTop = 32, kMostParts = 64;
// Logits a lane holds where the likeliest are asked for: few where there are few rows, whose parts
// are then more (8 rows of 32000, 8 of each: 17 -> 9 us).
constexpr int kFewHeld = 8, kHeld = 32;
constexpr int kHeldPart = 256 * kHeld;
constexpr float kLn2 = 0.6931471805599453f;

struct ProbParams {
  const void* x;
  const void* tokens;
  float *logprob, *entropy, *stats;        // stats: max and log s of each row
  float* top_logprob;
  int64_t* top_token;
  float* sums;                             // [M][parts][3]: max, s, t
  uint2* lists;                            // [M][parts][top]: key, index
  const float *dlogprob, *dentropy;        // backward
  void* dx;
  int64_t M, sx, sdx;
  int V, top, wide, parts, length;         // parts of a row and their logits
};

__device__ __forceinline__ int64_t token_of(const ProbParams& p, int64_t m) {
  return p.wide ? static_cast<const int64_t*>(p.tokens)[m] : static_cast<const int32_t*>(p.tokens)[m];
}

// 16 bytes of logits, or one where rows are not aligned to that.
template <typename T, bool VEC>
struct Logits {
  static constexpr int kElems = VEC ? 16 / (int)sizeof(T) : 1;
  static __device__ __forceinline__ void load(const T* src, float (&x)[kElems]) {
    if constexpr (!VEC) {
      x[0] = (float)src[0];
    } else {
      const u4v q = *reinterpret_cast<const u4v*>(src);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
          x[2 * i] = __uint_as_float(q[i] << 16);
          x[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
        } else {
          x[i] = __uint_as_float(q[i]);
        }
      }
    }
  }
  static __device__ __forceinline__ void store(T* dst, const float (&x)[kElems]) {
    if constexpr (!VEC) {
      dst[0] = (T)x[0];
    } else {
      u4v q;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
          typedef float f2v __attribute__((ext_vector_type(2)));
          typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
          q[i] = __builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{x[2 * i], x[2 * i + 1]}), bf2v));
        } else {
          q[i] = __float_as_uint(x[i]);
        }
      }
      *reinterpret_cast<u4v*>(dst) = q;
    }
  }
};

// The running maximum, and s and t relative to it.
struct Sums {
  float m, s, t;
};
__device__ __forceinline__ float finite_max(float m) { return m == -__builtin_inff() ? 0.0f : m; }
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }
// d exp d, where e = exp d: 0 for d = -infinity, NaN for a NaN.
__device__ __forceinline__ float add_entropy(float d, float e, float t) { return __builtin_fmaf(__builtin_fmaxf(d, -200.0f), e, t); }
__device__ __forceinline__ void raise(Sums& a, float m) {
  if (m > a.m) {
    const float d = finite_max(a.m) - m, r = a.m == -__builtin_inff() ? 0.0f : exp_of(d);
    a.t = a.s != 0.0f ? __builtin_fmaf(__builtin_fmaxf(d, -200.0f), a.s, a.t) * r : 0.0f;
    a.s *= r;
    a.m = m;
  }
}
__device__ __forceinline__ Sums both(Sums a, Sums b) {
  const float m = __builtin_fmaxf(a.m, b.m);
  raise(a, m);
  raise(b, m);
  return Sums{m, a.s + b.s, a.t + b.t};
}
template <int D>
__device__ __forceinline__ Sums with_lane(const Sums& a) {
  const Sums o{lane_xor_c<D>(a.m), lane_xor_c<D>(a.s), lane_xor_c<D>(a.t)};
  return (__lane_id() & D) ? both(o, a) : both(a, o);  // the same order in both lanes of a pair
}
__device__ __forceinline__ Sums over_wave(Sums a) {
  a = with_lane<1>(a);
  a = with_lane<2>(a);
  a = with_lane<4>(a);
  a = with_lane<8>(a);
  a = with_lane<16>(a);
  return with_lane<32>(a);
}

// What a row's sums say, from one thread.
template <typename T>
__device__ __forceinline__ void finish(const ProbParams& p, int64_t row, const Sums& a) {
  const bool none = a.m == -__builtin_inff() && a.s == 0.0f;  // every logit is -infinity
  const float logs = __builtin_amdgcn_logf(a.s) * kLn2;
  p.entropy[row] = none ? 0.0f : logs - a.t / a.s;
  if (p.stats != nullptr) {
    p.stats[2 * row] = a.m;
    p.stats[2 * row + 1] = logs;
  }
  const int64_t v = token_of(p, row);
  float r = v < 0 ? 0.0f : __builtin_nanf("");
  if (v >= 0 && v < p.V) r = none ? -__builtin_inff() : ((float)(static_cast<const T*>(p.x) + row * p.sx)[v] - a.m) - logs;
  p.logprob[row] = r;
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void prob_fwd_kernel(ProbParams p) {
  typedef Logits<T, VEC> L;
  __shared__ Sums waves[4];
  const int64_t row = blockIdx.x / p.parts;
  const int part = (int)(blockIdx.x - row * p.parts), from = part * p.length, to = min(p.V, from + p.length);
  const T* x = static_cast<const T*>(p.x) + row * p.sx;
  Sums a{-__builtin_inff(), 0.0f, 0.0f};
#pragma unroll 2
  for (int v = from + (int)threadIdx.x * L::kElems; v < to; v += 256 * L::kElems) {
    float e[L::kElems];
    L::load(x + v, e);
    float m = e[0];
#pragma unroll
    for (int i = 1; i < L::kElems; ++i) m = __builtin_fmaxf(m, e[i]);
    raise(a, m);
    const float ref = finite_max(a.m);
#pragma unroll
    for (int i = 0; i < L::kElems; ++i) {
      const float d = e[i] - ref, w = exp_of(d);
      a.s += w;
      a.t = add_entropy(d, w, a.t);
    }
  }
  a = over_wave(a);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = a;
  __syncthreads();
  if (threadIdx.x != 0) return;
  a = both(both(waves[0], waves[1]), both(waves[2], waves[3]));
  if (p.parts == 1) {
    finish<T>(p, row, a);
  } else {
    float* out = p.sums + 3 * (int64_t)blockIdx.x;
    out[0] = a.m;
    out[1] = a.s;
    out[2] = a.t;
  }
}

// A word that sorts as the logits do: NaN first, then +infinity down to -infinity; 0 is less than any.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = x != x ? 0x7fc00000u : __float_as_uint(x + 0.0f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
template <int D>
__device__ __forceinline__ uint32_t max_with_lane(uint32_t x) {
  return max(x, __float_as_uint(lane_xor_c<D>(__uint_as_float(x))));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max_with_lane<1>(x);
  x = max_with_lane<2>(x);
  x = max_with_lane<4>(x);
  x = max_with_lane<8>(x);
  x = max_with_lane<16>(x);
  return max_with_lane<32>(x);
}
// The largest key over the wave, of equal ones the lowest index.
__device__ __forceinline__ uint2 best_of_wave(uint2 a) {
  const uint32_t k = wave_max(a.x);
  return uint2{k, ~wave_max(a.x == k ? ~a.y : 0u)};
}

template <typename T, bool VEC, int HELD>
__global__ __launch_bounds__(256) void prob_top_kernel(ProbParams p) {
  typedef Logits<T, VEC> L;
  constexpr int kLoads = HELD / L::kElems;
  __shared__ Sums waves[4];
  __shared__ uint2 lists[4][kMostTop];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x / p.parts;
  const int part = (int)(blockIdx.x - row * p.parts), from = part * p.length, to = min(p.V, from + p.length);
  const T* x = static_cast<const T*>(p.x) + row * p.sx;
  float e[kLoads][L::kElems];
  float m = -__builtin_inff();
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    const int v = from + (k * 256 + (int)threadIdx.x) * L::kElems;
#pragma unroll
    for (int i = 0; i < L::kElems; ++i) e[k][i] = -__builtin_inff();
    if (v < to) L::load(x + v, e[k]);
#pragma unroll
    for (int i = 0; i < L::kElems; ++i) m = __builtin_fmaxf(m, e[k][i]);
  }
  Sums a{m, 0.0f, 0.0f};
  const float ref = finite_max(m);
  uint32_t key[kLoads][L::kElems];
#pragma unroll
  for (int k = 0; k < kLoads; ++k) {
    const int v = from + (k * 256 + (int)threadIdx.x) * L::kElems;
#pragma unroll
    for (int i = 0; i < L::kElems; ++i) {
      const float d = e[k][i] - ref, w = exp_of(d);
      a.s += w;
      a.t = add_entropy(d, w, a.t);
      key[k][i] = v < to ? key_of(e[k][i]) : 0u;
    }
  }
  a = over_wave(a);
  if (lane == 0) waves[wave] = a;
  for (int r = 0; r < p.top; ++r) {
    uint2 best{0u, 0xffffffffu};
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
#pragma unroll
      for (int i = 0; i < L::kElems; ++i)
        if (key[k][i] > best.x) best = uint2{key[k][i], (uint32_t)(from + (k * 256 + (int)threadIdx.x) * L::kElems + i)};
    best = best_of_wave(best);
    if (lane == 0) lists[wave][r] = best;
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
#pragma unroll
      for (int i = 0; i < L::kElems; ++i)
        if (best.y == (uint32_t)(from + (k * 256 + (int)threadIdx.x) * L::kElems + i)) key[k][i] = 0u;
  }
  __syncthreads();
  if (wave != 0) return;
  if (lane == 0) {
    a = both(both(waves[0], waves[1]), both(waves[2], waves[3]));
    float* out = p.sums + 3 * (int64_t)blockIdx.x;
    out[0] = a.m;
    out[1] = a.s;
    out[2] = a.t;
  }
  int at = 0;
  for (int r = 0; r < p.top; ++r) {
    const uint2 head = lane < 4 && at < p.top ? lists[lane][at] : uint2{0u, 0xffffffffu};
    const uint2 best = best_of_wave(head);
    if (lane < 4 && head.y == best.y) ++at;
    if (lane == 0) p.lists[(int64_t)blockIdx.x * p.top + r] = best;
  }
}

// A wave a row: joins its parts, and merges their lists (a lane a part).
template <typename T>
__global__ __launch_bounds__(64) void prob_join_kernel(ProbParams p) {
  __shared__ uint2 lists[kMostParts][kMostTop];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const float* src = p.sums + 3 * row * p.parts;
  Sums a{-__builtin_inff(), 0.0f, 0.0f};
  if (lane < p.parts) a = Sums{src[3 * lane], src[3 * lane + 1], src[3 * lane + 2]};
  a = over_wave(a);
  if (lane == 0) finish<T>(p, row, a);
  if (p.top == 0) return;
  for (int i = lane; i < p.parts * p.top; i += 64) lists[i / p.top][i % p.top] = p.lists[row * p.parts * p.top + i];
  __syncthreads();
  const float logs = __builtin_amdgcn_logf(a.s) * kLn2;
  int at = 0;
  for (int r = 0; r < p.top; ++r) {
    const uint2 head = lane < p.parts && at < p.top ? lists[lane][at] : uint2{0u, 0xffffffffu};
    const uint2 best = best_of_wave(head);
    if (head.y == best.y) ++at;
    if (lane == 0) {
      p.top_token[row * p.top + r] = best.y;
      const float x = logit_of(best.x);
      p.top_logprob[row * p.top + r] = x == -__builtin_inff() && a.m == a.m && a.s == a.s ? x : (x - a.m) - logs;
    }
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void prob_bwd_kernel(ProbParams p) {
  typedef Logits<T, VEC> L;
  const int64_t row = blockIdx.x / p.parts;
  const int part = (int)(blockIdx.x - row * p.parts), from = part * p.length, to = min(p.V, from + p.length);
  const T* x = static_cast<const T*>(p.x) + row * p.sx;
  T* dx = static_cast<T*>(p.dx) + row * p.sdx;
  const float m = p.stats[2 * row], logs = p.stats[2 * row + 1];
  const int64_t token = token_of(p, row);
  const float g = p.dlogprob != nullptr && token >= 0 && token < p.V ? p.dlogprob[row] : 0.0f;
  const float ge = p.dentropy != nullptr ? p.dentropy[row] : 0.0f;
  // every logit is -infinity, or no gradient comes (a row of padding), whatever the logits are
  const bool none = (m == -__builtin_inff() && logs == -__builtin_inff()) || (g == 0.0f && ge == 0.0f);
  // dx = -p (g + ge (log p + entropy)), and g more at the token
  const float base = __builtin_fmaf(ge, p.entropy[row], g);
#pragma unroll 2
  for (int v = from + (int)threadIdx.x * L::kElems; v < to; v += 256 * L::kElems) {
    float e[L::kElems];
    L::load(x + v, e);
#pragma unroll
    for (int i = 0; i < L::kElems; ++i) {
      const float d = (e[i] - m) - logs;
      float r = -exp_of(d) * __builtin_fmaf(ge, __builtin_fmaxf(d, -200.0f), base);
      if (token == v + i) r += g;
      e[i] = none ? 0.0f : r;
    }
    L::store(dx + v, e);
  }
}

// ---- host ---------------------------------------------------------------------------

struct Plan {
  int parts, length;
  bool few;              // parts of 256 kFewHeld logits
  int64_t lists, total;  // offset of the lists
};
// A row a workgroup; parts of 2048 logits at least where there are fewer rows than fill the device (8 rows of 32000,
// forward and backward: 20.5 us in whole rows, 16.5 in parts; 64 rows 21.4 and 17.3).
// Where the likeliest are asked for, parts of what a workgroup's registers hold.
Plan make_plan(int64_t M, int64_t V, int64_t top) {
  Plan r;
  int64_t parts = std::max<int64_t>(1, std::min<int64_t>({512 / M, V / 2048, kMostParts}));
  r.few = false;
  if (top > 0) {
    const int64_t fine = (V + 256 * kFewHeld - 1) / (256 * kFewHeld);
    r.few = fine <= kMostParts && M * fine <= 4096;
    parts = r.few ? fine : (V + kHeldPart - 1) / kHeldPart;
  }
  r.length = (int)(((V + parts - 1) / parts + 63) / 64 * 64);
  r.parts = (int)((V + r.length - 1) / r.length);
  r.lists = align256(M * r.parts * 12);
  r.total = r.parts > 1 || top > 0 ? r.lists + align256(M * r.parts * top * 8) : 0;
  return r;
}

template <typename T>
void (*top_kernel(bool vec, bool few))(ProbParams) {
  if (few) return vec ? prob_top_kernel<T, true, kFewHeld> : prob_top_kernel<T, false, kFewHeld>;
  return vec ? prob_top_kernel<T, true, kHeld> : prob_top_kernel<T, false, kHeld>;
}

int check_sizes(const char* who, int64_t M, int64_t V, int64_t stride, int token_bits, int dtype) {
  if (M < 1 || V < 1) return set_error(GS_ERR_INVALID, "%s: M and V must be > 0; got M=%lld, V=%lld", who, (long long)M, (long long)V);
  if (M > (1ll << 23) || V > (1ll << 24))
    return set_error(GS_ERR_INVALID, "%s: M/V out of supported range (M=%lld, V=%lld)", who, (long long)M, (long long)V);
  if (token_bits != 32 && token_bits != 64)
    return set_error(GS_ERR_INVALID, "%s: tokens must have 32 or 64 bits; got %d", who, token_bits);
  if (stride < 0) return set_error(GS_ERR_INVALID, "%s: a negative row stride (%lld)", who, (long long)stride);
  return check_dtype(who, dtype);
}
int check_fwd(const gs_logprobs_args* a, const char* who) {
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  const int rc = check_sizes(who, a->M, a->V, a->sx, a->token_bits, a->dtype);
  if (rc) return rc;
  if (a->top < 0 || a->top > kMostTop || a->top > a->V)
    return set_error(GS_ERR_INVALID, "%s: top must be 0 to %d and at most V=%lld; got %lld", who, kMostTop, (long long)a->V,
                     (long long)a->top);
  if (a->top > 0 && a->V > (int64_t)kHeldPart * kMostParts)
    return set_error(GS_ERR_INVALID, "%s: top takes at most %d logits a row; got V=%lld", who, kHeldPart * kMostParts,
                     (long long)a->V);
  if (a->top > 0 && a->M * make_plan(a->M, a->V, a->top).parts >= (1ll << 24))
    return set_error(GS_ERR_INVALID, "%s: more workgroups than a launch holds (M=%lld, V=%lld)", who, (long long)a->M,
                     (long long)a->V);
  return GS_OK;
}

bool aligned16(const void* p, int64_t stride, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride * size % 16 == 0;
}
// Whole accesses of 16 bytes: aligned rows of a multiple of that.
bool whole(const void* p, int64_t stride, int64_t V, int size) { return aligned16(p, stride, size) && V * size % 16 == 0; }

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int64_t gs_logprobs_scratch_bytes(const gs_logprobs_args* a) {
  clear_error();
  const int rc = check_fwd(a, "gs_logprobs_scratch_bytes");
  return rc ? rc : make_plan(a->M, a->V, a->top).total;
}

extern "C" int gs_logprobs_fwd(const gs_logprobs_args* a, hipStream_t stream) {
  const char* who = "gs_logprobs_fwd";
  clear_error();
  int rc = check_fwd(a, who);
  if (rc) return rc;
  if (!a->x || !a->tokens || !a->logprob || !a->entropy || (a->top > 0 && (!a->top_logprob || !a->top_token)))
    return set_error(GS_ERR_INVALID, "%s: x, tokens, logprob, entropy (and with top its outputs) must be non-NULL device pointers", who);
  const Plan plan = make_plan(a->M, a->V, a->top);
  if ((rc = check_plain_scratch(who, a->scratch, a->scratch_bytes, plan.total))) return rc;
  ProbParams p{};
  p.x = a->x;
  p.tokens = a->tokens;
  p.logprob = a->logprob;
  p.entropy = a->entropy;
  p.stats = a->stats;
  p.top_logprob = a->top_logprob;
  p.top_token = a->top_token;
  p.sums = static_cast<float*>(a->scratch);
  p.lists = reinterpret_cast<uint2*>(static_cast<char*>(a->scratch) + plan.lists);
  p.M = a->M;
  p.sx = a->sx;
  p.V = (int)a->V;
  p.top = (int)a->top;
  p.wide = a->token_bits == 64;
  p.parts = plan.parts;
  p.length = plan.length;
  const int size = a->dtype == GS_DTYPE_F32 ? 4 : 2;
  const bool vec = whole(a->x, a->sx, a->V, size);
  void (*fn)(ProbParams);
  if (a->top > 0)
    fn = size == 4 ? top_kernel<float>(vec, plan.few) : top_kernel<__bf16>(vec, plan.few);
  else
    fn = size == 4 ? (vec ? prob_fwd_kernel<float, true> : prob_fwd_kernel<float, false>)
                   : (vec ? prob_fwd_kernel<__bf16, true> : prob_fwd_kernel<__bf16, false>);
  hipLaunchKernelGGL(fn, dim3((unsigned)(a->M * plan.parts)), dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  if (plan.parts > 1 || a->top > 0) {
    hipLaunchKernelGGL(size == 4 ? prob_join_kernel<float> : prob_join_kernel<__bf16>, dim3((unsigned)a->M), dim3(64), 0, stream, p);
    GS_CHECK_HIP(hipGetLastError());
  }
  return GS_OK;
}

extern "C" int gs_logprobs_bwd(const gs_logprobs_bwd_args* a, hipStream_t stream) {
  const char* who = "gs_logprobs_bwd";
  clear_error();
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  const int rc = check_sizes(who, a->M, a->V, a->sx, a->token_bits, a->dtype);
  if (rc) return rc;
  if (!a->x || !a->tokens || !a->entropy || !a->stats || !a->dx)
    return set_error(GS_ERR_INVALID, "%s: x, tokens, entropy, stats and dx must be non-NULL device pointers", who);
  if (a->M > 1 && a->sdx < a->V)
    return set_error(GS_ERR_INVALID, "%s: a row stride of %lld does not hold V=%lld", who, (long long)a->sdx, (long long)a->V);
  const Plan plan = make_plan(a->M, a->V, 0);
  ProbParams p{};
  p.x = a->x;
  p.tokens = a->tokens;
  p.entropy = const_cast<float*>(a->entropy);
  p.stats = const_cast<float*>(a->stats);
  p.dlogprob = a->dlogprob;
  p.dentropy = a->dentropy;
  p.dx = a->dx;
  p.M = a->M;
  p.sx = a->sx;
  p.sdx = a->sdx;
  p.V = (int)a->V;
  p.wide = a->token_bits == 64;
  p.parts = plan.parts;
  p.length = plan.length;
  const int size = a->dtype == GS_DTYPE_F32 ? 4 : 2;
  const bool vec = whole(a->x, a->sx, a->V, size) && aligned16(a->dx, a->sdx, size);
  void (*fn)(ProbParams) = size == 4 ? (vec ? prob_bwd_kernel<float, true> : prob_bwd_kernel<float, false>)
                                     : (vec ? prob_bwd_kernel<__bf16, true> : prob_bwd_kernel<__bf16, false>);
  hipLaunchKernelGGL(fn, dim3((unsigned)(a->M * plan.parts)), dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}
