// Linear with bias, activation and residual (gfx950): y = act(x w^T + bias) + residual
// and its gradients, in bf16 (gemm_bf16.hip) and fp32 (gemm.hip).
//
// Backward: dpre = dy act'(pre) and its column sums (dbias) in one pass over dy and
// pre, then dx = dpre w and dw = dpre^T x. In bf16 dpre is rounded to bf16, which is
// what the matrix instruction takes (the sums stay fp32; dbias sums the unrounded
// values). dw sums over all M rows: it is split over K where its tiles alone do not fill
// the device, and the splits' fp32 sums are added in order.
#include "gs_gemm_bf16.h"

namespace gs {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 128;  // rows of one workgroup of the dpre pass

typedef unsigned int u4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));

// V consecutive elements (16 bytes) at any alignment; those from `have` on are zeros.
template <typename T>
struct Wide;
template <>
struct Wide<float> {
  static constexpr int V = 4;
  static __device__ __forceinline__ void load(const float* p, int have, float (&x)[4]) {
    if (have >= 4) {
      const f4u w = *reinterpret_cast<const f4u*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = i < have ? p[i] : 0.0f;
    }
  }
  static __device__ __forceinline__ void store(float* p, int have, const float (&x)[4]) {
    if (have >= 4) {
      *reinterpret_cast<f4u*>(p) = f4u{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < have) p[i] = x[i];
    }
  }
};
template <>
struct Wide<__bf16> {
  static constexpr int V = 8;
  static __device__ __forceinline__ void load(const __bf16* p, int have, float (&x)[8]) {
    if (have >= 8) {
      const u4u w = *reinterpret_cast<const u4u*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = i < have ? (float)p[i] : 0.0f;
    }
  }
  static __device__ __forceinline__ void store(__bf16* p, int have, const float (&x)[8]) {
    if (have >= 8) {
      u4u w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = __builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{x[2 * i], x[2 * i + 1]}), bf2v));
      *reinterpret_cast<u4u*>(p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < have) p[i] = (__bf16)x[i];
    }
  }
};

struct DpreArgs {
  const void* pre;  // NULL: no activation, only the column sums
  const void* dy;
  void* dpre;       // contiguous, or NULL (column sums only)
  float* part;      // [ceil(M / kRows)][N], or NULL
  int64_t sdy;
  int M, N, act;
};

// A workgroup takes 16 lanes of columns (16 bytes each) by kRows rows; its 16 row lanes
// take every 16th row, four at a time, and their sums are joined through LDS in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void dpre_kernel(DpreArgs p) {
  constexpr int V = Wide<T>::V, kAhead = 4;
  __shared__ float red[16][16 * V + 1];
  const int jl = threadIdx.x & 15, rl = threadIdx.x >> 4, j = (blockIdx.x * 16 + jl) * V;
  const int r0 = blockIdx.y * kRows, r1 = min(p.M, r0 + kRows), have = p.N - j;
  float sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) sum[v] = 0.0f;
  if (have > 0) {
    const T* dy = static_cast<const T*>(p.dy) + j;
    const T* pre = static_cast<const T*>(p.pre) + j;
    T* dpre = static_cast<T*>(p.dpre) + j;
    for (int r = r0 + rl; r < r1; r += 16 * kAhead) {
      float d[kAhead][V], x[kAhead][V];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int q = r + 16 * u;
        Wide<T>::load(dy + q * p.sdy, q < r1 ? have : 0, d[u]);
        if (p.pre != nullptr) Wide<T>::load(pre + (int64_t)q * p.N, q < r1 ? have : 0, x[u]);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int q = r + 16 * u;
        if (p.pre != nullptr) {
          act_slopes(x[u], p.act);
#pragma unroll
          for (int v = 0; v < V; ++v) d[u][v] *= x[u][v];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] += d[u][v];
        if (p.dpre != nullptr && q < r1) Wide<T>::store(dpre + (int64_t)q * p.N, have, d[u]);
      }
    }
  }
  if (p.part == nullptr) return;
#pragma unroll
  for (int v = 0; v < V; ++v) red[rl][jl * V + v] = sum[v];
  __syncthreads();
  const int c = threadIdx.x, col = blockIdx.x * 16 * V + c;
  if (c < 16 * V && col < p.N) {
    float s = red[0][c];
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][c];
    p.part[(int64_t)blockIdx.y * p.N + col] = s;
  }
}

// dst[e] = sum over parts of src[part * n + e], rounded to the tensor's type: a workgroup
// takes 16 columns, its 16 part lanes every 16th part, joined through LDS in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void sum_columns_kernel(T* dst, const float* src, int n, int parts) {
  __shared__ float red[16][17];
  const int c = threadIdx.x & 15, l = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
  float s = 0.0f;
  if (e < n)
    for (int k = l; k < parts; k += 16) s += src[(int64_t)k * n + e];
  red[l][c] = s;
  __syncthreads();
  if (l == 0 && e < n) {
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][c];
    dst[e] = (T)s;
  }
}

// fp32: what follows the product's sums (with the bias already added), in place in y.
struct PostArgs {
  float* y;
  int64_t ldy;
  LinearEpilogue e;
  int64_t n;
  int N;
};
__global__ __launch_bounds__(kThreads) void post_kernel(PostArgs p) {
  for (int64_t e = blockIdx.x * (int64_t)kThreads + threadIdx.x; e < p.n; e += (int64_t)gridDim.x * kThreads) {
    const int64_t i = e / p.N;
    const int j = (int)(e - i * p.N);
    float x = p.y[i * p.ldy + j];
    if (p.e.pre != nullptr) static_cast<float*>(p.e.pre)[e] = x;
    float v[1] = {x};
    act_values(v, p.e.act);
    x = v[0];
    if (p.e.residual != nullptr) x += static_cast<const float*>(p.e.residual)[i * p.e.ldr + j];
    p.y[i * p.ldy + j] = x;
  }
}

int check_linear(const char* who, int64_t M, int64_t N, int64_t K, int dtype, int act) {
  if (M < 1 || N < 1 || K < 1)
    return set_error(GS_ERR_INVALID, "%s: M, N and K must be > 0; got %lld, %lld, %lld", who, (long long)M,
                     (long long)N, (long long)K);
  if (M > INT32_MAX / 2 || N > (1 << 24) || K > (1 << 24))
    return set_error(GS_ERR_INVALID, "%s: sizes out of supported range (M=%lld, N=%lld, K=%lld)", who, (long long)M,
                     (long long)N, (long long)K);
  if (dtype != GS_DTYPE_F32 && dtype != GS_DTYPE_BF16)
    return set_error(GS_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
  if (act < GS_ACT_NONE || act > GS_ACT_SIGMOID) return set_error(GS_ERR_INVALID, "%s: unknown activation %d", who, act);
  return GS_OK;
}

int check_scratch(const char* who, const void* scratch, int64_t bytes, int64_t need) {
  if (need > 0 && (scratch == nullptr || bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 255u) != 0))
    return set_error(GS_ERR_INVALID, "%s: scratch of %lld bytes, 256-byte aligned, required; got %lld at %p", who,
                     (long long)need, (long long)bytes, scratch);
  return GS_OK;
}

int check_fwd(const gs_linear_args* a, const char* who) {
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  const int rc = check_linear(who, a->M, a->N, a->K, a->dtype, a->activation);
  if (rc) return rc;
  if ((a->M > 1 && (a->sy < a->N || a->sx < 0 || a->sr < 0)))
    return set_error(GS_ERR_INVALID, "%s: row strides (x %lld, residual %lld, y %lld) do not describe M rows", who,
                     (long long)a->sx, (long long)a->sr, (long long)a->sy);
  return GS_OK;
}

int check_bwd(const gs_linear_bwd_args* a, const char* who) {
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  const int rc = check_linear(who, a->M, a->N, a->K, a->dtype, a->activation);
  if (rc) return rc;
  if (a->M > 1 && (a->sx < 0 || a->sdy < 0))
    return set_error(GS_ERR_INVALID, "%s: row strides (x %lld, dy %lld) do not describe M rows", who, (long long)a->sx,
                     (long long)a->sdy);
  return GS_OK;
}

int fwd_split(const gs_linear_args* a) {
  return a->dtype == GS_DTYPE_BF16 ? gemm_bf16_pick_split((int)a->M, (int)a->N, (int)a->K) : 1;
}

int64_t fwd_scratch(const gs_linear_args* a) {
  const int s = fwd_split(a);
  return s > 1 ? align256(s * a->M * a->N * 4) : 0;
}

// The backward's scratch: dpre, the column sums' parts, the splits of dx and of dw.
struct BwdPlan {
  int split_x, split_w;
  int64_t dpre, cols, dx, dw, total;  // byte offsets; -1: not used
};

BwdPlan bwd_plan(const gs_linear_bwd_args* a) {
  BwdPlan p{};
  const bool bf16 = a->dtype == GS_DTYPE_BF16;
  const int64_t size = bf16 ? 2 : 4;
  p.split_x = bf16 ? gemm_bf16_pick_split((int)a->M, (int)a->K, (int)a->N) : 1;
  p.split_w = bf16 ? gemm_bf16_pick_split((int)a->N, (int)a->K, (int)a->M) : gemm_pick_split((int)a->N, (int)a->K, (int)a->M);
  int64_t at = 0;
  auto take = [&](bool used, int64_t bytes) {
    if (!used) return int64_t(-1);
    const int64_t r = at;
    at += align256(bytes);
    return r;
  };
  p.dpre = take(a->activation != GS_ACT_NONE && (a->dx || a->dw), a->M * a->N * size);
  p.cols = take(a->dbias != nullptr, (a->M + kRows - 1) / kRows * a->N * 4);
  p.dx = take(a->dx != nullptr && p.split_x > 1, p.split_x * a->M * a->K * 4);
  p.dw = take(a->dw != nullptr && p.split_w > 1, p.split_w * a->N * a->K * 4);
  p.total = at;
  return p;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int64_t gs_linear_scratch_bytes(const gs_linear_args* a) {
  clear_error();
  const int rc = check_fwd(a, "gs_linear_scratch_bytes");
  return rc ? rc : fwd_scratch(a);
}

extern "C" int gs_linear_fwd(const gs_linear_args* a, hipStream_t stream) {
  const char* who = "gs_linear_fwd";
  clear_error();
  int rc = check_fwd(a, who);
  if (rc) return rc;
  if (!a->x || !a->w || !a->y) return set_error(GS_ERR_INVALID, "%s: x, w and y must be non-NULL device pointers", who);
  if ((rc = check_scratch(who, a->scratch, a->scratch_bytes, fwd_scratch(a)))) return rc;
  LinearEpilogue e;
  e.bias = a->bias;
  e.residual = a->residual;
  e.pre = a->pre;
  e.ldr = a->sr;
  e.act = a->activation;
  if (a->dtype == GS_DTYPE_BF16) {
    GemmBf16Args g;
    g.a = static_cast<const __bf16*>(a->x);
    g.lda = a->sx;
    g.b = static_cast<const __bf16*>(a->w);
    g.ldb = a->K;
    g.y = static_cast<__bf16*>(a->y);
    g.ldy = a->sy;
    g.part = static_cast<float*>(a->scratch);
    g.epi = e;
    g.M = (int)a->M;
    g.N = (int)a->N;
    g.K = (int)a->K;
    g.ksplit = fwd_split(a);
    return gemm_bf16(g, stream, who);
  }
  GemmArgs g;
  g.a = static_cast<const float*>(a->x);
  g.lda = a->sx;
  g.b = static_cast<const float*>(a->w);
  g.ldb = a->K;
  g.c = static_cast<float*>(a->y);
  g.ldc = a->sy;
  g.bias = static_cast<const float*>(a->bias);
  g.M = (int)a->M;
  g.N = (int)a->N;
  g.K = (int)a->K;
  if ((rc = gemm_f32(g, stream, who))) return rc;
  if (e.act == GS_ACT_NONE && e.residual == nullptr && e.pre == nullptr) return GS_OK;
  PostArgs p{static_cast<float*>(a->y), a->sy, e, a->M * a->N, (int)a->N};
  hipLaunchKernelGGL(post_kernel, dim3((unsigned)std::min<int64_t>((p.n + kThreads - 1) / kThreads, 8192)),
                     dim3(kThreads), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}

extern "C" int64_t gs_linear_bwd_scratch_bytes(const gs_linear_bwd_args* a) {
  clear_error();
  const int rc = check_bwd(a, "gs_linear_bwd_scratch_bytes");
  return rc ? rc : bwd_plan(a).total;
}

extern "C" int gs_linear_bwd(const gs_linear_bwd_args* a, hipStream_t stream) {
  const char* who = "gs_linear_bwd";
  clear_error();
  int rc = check_bwd(a, who);
  if (rc) return rc;
  const bool act = a->activation != GS_ACT_NONE;
  if (!a->dy || (a->dx && !a->w) || (a->dw && !a->x) || (act && !a->pre))
    return set_error(GS_ERR_INVALID, "%s: dy, w (for dx), x (for dw) and pre (with an activation) must be non-NULL device pointers",
                     who);
  const BwdPlan plan = bwd_plan(a);
  if ((rc = check_scratch(who, a->scratch, a->scratch_bytes, plan.total))) return rc;
  char* scratch = static_cast<char*>(a->scratch);
  auto at = [&](int64_t off) -> void* { return off < 0 ? nullptr : scratch + off; };
  const bool bf16 = a->dtype == GS_DTYPE_BF16;
  const int chunks = (int)((a->M + kRows - 1) / kRows);
  if (plan.dpre >= 0 || plan.cols >= 0) {
    DpreArgs p{act ? a->pre : nullptr, a->dy, at(plan.dpre), static_cast<float*>(at(plan.cols)), a->sdy, (int)a->M,
               (int)a->N, a->activation};
    for (int first = 0; first < chunks; first += 65535) {  // grid.y
      DpreArgs q = p;
      const int64_t r = (int64_t)first * kRows;
      const int64_t size = bf16 ? 2 : 4;
      q.M = (int)std::min<int64_t>(a->M - r, 65535ll * kRows);
      if (q.pre) q.pre = static_cast<const char*>(q.pre) + r * a->N * size;
      q.dy = static_cast<const char*>(q.dy) + r * a->sdy * size;
      if (q.dpre) q.dpre = static_cast<char*>(q.dpre) + r * a->N * size;
      if (q.part) q.part += (int64_t)first * a->N;
      auto fn = bf16 ? dpre_kernel<__bf16> : dpre_kernel<float>;
      const int cols = bf16 ? 128 : 64;
      hipLaunchKernelGGL(fn, dim3((unsigned)((a->N + cols - 1) / cols), (unsigned)((q.M + kRows - 1) / kRows)), dim3(kThreads),
                         0, stream, q);
      GS_CHECK_HIP(hipGetLastError());
    }
  }
  const void* dpre = plan.dpre >= 0 ? at(plan.dpre) : a->dy;
  const int64_t sd = plan.dpre >= 0 ? a->N : a->sdy;
  if (a->dx != nullptr) {
    if (bf16) {
      GemmBf16Args g;
      g.a = static_cast<const __bf16*>(dpre);
      g.lda = sd;
      g.b = static_cast<const __bf16*>(a->w);
      g.ldb = a->K;
      g.y = static_cast<__bf16*>(a->dx);
      g.ldy = a->K;
      g.part = static_cast<float*>(at(plan.dx));
      g.M = (int)a->M;
      g.N = (int)a->K;
      g.K = (int)a->N;
      g.ksplit = plan.split_x;
      g.layout = kGemmNN;
      rc = gemm_bf16(g, stream, who);
    } else {
      GemmArgs g;
      g.a = static_cast<const float*>(dpre);
      g.lda = sd;
      g.b = static_cast<const float*>(a->w);
      g.ldb = a->K;
      g.c = static_cast<float*>(a->dx);
      g.ldc = a->K;
      g.M = (int)a->M;
      g.N = (int)a->K;
      g.K = (int)a->N;
      g.layout = kGemmNN;
      rc = gemm_f32(g, stream, who);
    }
    if (rc) return rc;
  }
  if (a->dw != nullptr) {
    if (bf16) {
      GemmBf16Args g;
      g.a = static_cast<const __bf16*>(dpre);
      g.lda = sd;
      g.b = static_cast<const __bf16*>(a->x);
      g.ldb = a->sx;
      g.y = static_cast<__bf16*>(a->dw);
      g.ldy = a->K;
      g.part = static_cast<float*>(at(plan.dw));
      g.M = (int)a->N;
      g.N = (int)a->K;
      g.K = (int)a->M;
      g.ksplit = plan.split_w;
      g.layout = kGemmTN;
      rc = gemm_bf16(g, stream, who);
    } else {
      GemmArgs g;
      g.a = static_cast<const float*>(dpre);
      g.lda = sd;
      g.b = static_cast<const float*>(a->x);
      g.ldb = a->sx;
      g.c = plan.dw >= 0 ? static_cast<float*>(at(plan.dw)) : static_cast<float*>(a->dw);
      g.ldc = a->K;
      g.split_stride = a->N * a->K;
      g.M = (int)a->N;
      g.N = (int)a->K;
      g.K = (int)a->M;
      g.ksplit = plan.split_w;
      g.layout = kGemmTN;
      rc = gemm_f32(g, stream, who);
      if (!rc && plan.dw >= 0)
        rc = sum_partials(static_cast<float*>(a->dw), g.c, a->N * a->K, plan.split_w, a->N * a->K, stream, who);
    }
    if (rc) return rc;
  }
  if (a->dbias != nullptr) {
    const float* part = static_cast<const float*>(at(plan.cols));
    const dim3 grid((unsigned)((a->N + 15) / 16));
    if (bf16)
      hipLaunchKernelGGL(sum_columns_kernel<__bf16>, grid, dim3(kThreads), 0, stream, static_cast<__bf16*>(a->dbias),
                         part, (int)a->N, chunks);
    else
      hipLaunchKernelGGL(sum_columns_kernel<float>, grid, dim3(kThreads), 0, stream, static_cast<float*>(a->dbias),
                         part, (int)a->N, chunks);
    GS_CHECK_HIP(hipGetLastError());
  }
  return rc;
}
