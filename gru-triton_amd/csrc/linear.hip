// Linear with bias, activation and residual (gfx950): y = act(x w^T + bias) + residual
// and its gradients, in bf16 (gemm_bf16.hip) and fp32 (gemm.hip).
//
// Backward: dpre = dy act'(pre) and its column sums (dbias) in one pass over dy and
// pre, then dx = dpre w and dw = dpre^T x. In bf16 dpre is rounded to bf16, which is
// what the matrix instruction takes (the sums stay fp32; dbias sums the unrounded
// values): it takes dx and dw from 0.00166 of their size off 64 bits, which is their own
// rounding, to 0.00235. pre is kept in 16 bits (gs_gemm_bf16.h). dw sums over all M rows: it is split over K where its tiles alone do not fill
// the device, and the splits' fp32 sums are added in order. Small backward products go in
// one launch (gemm_bf16_pair, gemm_pair).
//
// Time on the GPU of a training step's kernels, in us (the products' own comments say what
// bounds them; the dpre pass reads dy, and pre where there is an activation, at 3.9 TB/s):
//   M, N, K                    forward  dpre  dx    dw    sums joined
//   2048, 1024, 512 bf16 gelu  11.4     6.4   15.1 together
//   32768, 2048, 1024 bf16     170      35    132   110   19
//   1650, 1002, 301 fp32 silu  26       8     39 together 4.1
#include "gs_gemm_bf16.h"

namespace gs {
namespace {

constexpr int kThreads = 256;

// Rows of one workgroup of the dpre pass: as many workgroups as fill the device several
// times over, from 16 rows (a row for each of its lanes) to 128 (M = 2048, N = 1024 in
// bf16: 13.5 us in 128 workgroups of 128 rows, 5 in 1024 of 16).
int64_t dpre_rows(int64_t M, int64_t N, bool bf16) {
  const int64_t across = (N + (bf16 ? 127 : 63)) / (bf16 ? 128 : 64);
  int64_t rows = 16;
  while (rows < 128 && (M + rows - 1) / rows * across > 2048) rows *= 2;
  return rows;
}

typedef float f2v __attribute__((ext_vector_type(2)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));

// 16 bytes of a row at any alignment: `have` elements exist from p on (the rest reads as
// zeros, and is not written) and `before` elements of the row in front of it.
template <typename T>
struct Wide;
template <>
struct Wide<float> {
  static constexpr int V = 4;
  typedef f4u Raw;
  static __device__ __forceinline__ Raw load(const float* p, int have, int) {
    if (have >= 4) return *reinterpret_cast<const f4u*>(p);
    f4u w = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < have) w[i] = p[i];
    return w;
  }
  static __device__ __forceinline__ void values(const Raw& w, int, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = w[i];
  }
  static __device__ __forceinline__ void kept(const Raw& w, int have, float (&x)[4]) { values(w, have, x); }  // of pre
  static __device__ __forceinline__ void store(float* p, int have, const float (&x)[4]) {
    if (have >= 4) {
      *reinterpret_cast<f4u*>(p) = f4u{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i < have) p[i] = x[i];
    }
  }
};
template <>
struct Wide<__bf16> {
  static constexpr int V = 8;
  typedef Granule Raw;
  static __device__ __forceinline__ Raw load(const __bf16* p, int have, int before) {
    return granule_load(p, have, before);
  }
  static __device__ __forceinline__ void values(const Raw& w, int have, float (&x)[8]) {
    granule_floats(granule_settle(w, have), x);
  }
  static __device__ __forceinline__ void kept(const Raw& w, int have, float (&x)[8]) {
    kept_floats(granule_settle(w, have), x);
  }
  static __device__ __forceinline__ void store(__bf16* p, int have, const float (&x)[8]) {
    if (have >= 8) {
      GranuleAt w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = __builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{x[2 * i], x[2 * i + 1]}), bf2v));
      *reinterpret_cast<GranuleAt*>(p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < have) p[i] = (__bf16)x[i];
    }
  }
};

struct DpreArgs {
  const void* pre;  // NULL: no activation, only the column sums
  const void* dy;
  void* dpre;       // row stride ldp >= N, zeros from column N on; or NULL (column sums only)
  float* part;      // [ceil(M / rows)][N], or NULL
  int64_t sdy, ldp;
  int M, N, act, rows;
};

// A workgroup takes 16 lanes of columns (16 bytes each) by `rows` rows; its 16 row lanes
// take every 16th row, four at a time, and their sums are joined through LDS in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void dpre_kernel(DpreArgs p) {
  constexpr int V = Wide<T>::V, kAhead = 4;
  __shared__ float red[16][16 * V + 1];
  const int jl = threadIdx.x & 15, rl = threadIdx.x >> 4, j = (blockIdx.x * 16 + jl) * V;
  const int r0 = blockIdx.y * p.rows, r1 = min(p.M, r0 + p.rows), have = p.N - j;
  float sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) sum[v] = 0.0f;
  if (have > 0) {
    const T* dy = static_cast<const T*>(p.dy) + j;
    const T* pre = static_cast<const T*>(p.pre) + j;
    T* dpre = static_cast<T*>(p.dpre) + j;
    // INSIDE: whole columns and rows, no load under a mask
    auto run = [&](auto INSIDE) __attribute__((always_inline)) {
      constexpr bool in = decltype(INSIDE)::value;
      for (int r = r0 + rl; r < r1; r += 16 * kAhead) {
        typename Wide<T>::Raw rd[kAhead], rx[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int q = min(r + 16 * u, r1 - 1);  // past the end: a row of its own again, not used
          const int h = in ? V : have;
          rd[u] = Wide<T>::load(dy + q * p.sdy, h, in ? 0 : j);
          if (p.pre != nullptr) rx[u] = Wide<T>::load(pre + (int64_t)q * p.N, h, in ? 0 : j);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int q = r + 16 * u;
          if (q >= r1) break;
          const int h = in ? V : have;
          float d[V], x[V];
          Wide<T>::values(rd[u], h, d);
          if (p.pre != nullptr) {
            Wide<T>::kept(rx[u], h, x);
            act_slopes(x, p.act);
#pragma unroll
            for (int v = 0; v < V; ++v) d[v] *= x[v];
          }
#pragma unroll
          for (int v = 0; v < V; ++v) sum[v] += d[v];
          if (p.dpre != nullptr) Wide<T>::store(dpre + q * p.ldp, in ? V : min(V, (int)p.ldp - j), d);
        }
      }
    };
    if ((int)(blockIdx.x + 1) * 16 * V <= p.N)  // uniform
      run(std::true_type{});
    else
      run(std::false_type{});
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

// Rows of bf16 operands copied to rows of whole 16-byte granules, zeros from `cols` on,
// so that the product can take them straight to LDS.
struct PadJob {
  const __bf16* src;
  __bf16* dst;
  int64_t ld, octets;  // octets: rows * ldp / 8; 0: no job
  int cols, ldp;
};
__global__ __launch_bounds__(kThreads) void pad_kernel(PadJob a, PadJob b) {
  const int64_t all = a.octets + b.octets, step = (int64_t)gridDim.x * kThreads;
  constexpr int kAhead = 4;
  for (int64_t q0 = blockIdx.x * (int64_t)kThreads + threadIdx.x; q0 < all; q0 += kAhead * step) {
    Granule w[kAhead];
    int have[kAhead];
    auto at = [&](int u, const PadJob** p) {  // the granule's job and its place there
      const int64_t q = q0 + u * step;
      *p = q < a.octets ? &a : &b;
      return q < a.octets ? q : q - a.octets;
    };
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (q0 + u * step >= all) continue;
      const PadJob* p;
      const int64_t o = at(u, &p);
      const int per = p->ldp / 8;
      const int64_t row = o / per;
      const int c = (int)(o - row * per) * 8;
      have[u] = p->cols - c;
      w[u] = granule_load(p->src + row * p->ld + c, have[u], c);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (q0 + u * step >= all) continue;
      const PadJob* p;
      const int64_t o = at(u, &p);
      *reinterpret_cast<Granule*>(p->dst + o * 8) = granule_settle(w[u], have[u]);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sum_columns_kernel(ColumnSums c) {
  __shared__ float red[16][17];
  sum_columns<T>(c, blockIdx.x, red);
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

// bf16 products of this many operations and more copy operands whose rows are not whole
// 16-byte granules. x w^T and dpre w go well through registers (M = 10000, N = 501,
// K = 333, 3.3 GFLOP: 19.5 us, 23.0 with copies; 13977 x 3171 x 694, 62 GFLOP: 141 and
// 102). dpre^T x, whose rows all start at another alignment and which is split, does not
// (M = 600, N = 501, K = 333, 0.2 GFLOP: 16.6 and 13.6 us; 20000 x 1021 x 515: 212 and 70);
// its copy of dpre then serves dx too.
constexpr double kPadFlops = 8e9, kPadFlopsDw = 0.2e9;

int64_t up8(int64_t x) { return (x + 7) / 8 * 8; }

// Rows of `n` bf16 that a product could take straight to LDS.
bool granular(const void* p, int64_t ld, int64_t n) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0 && n % 8 == 0;
}

// Scratch laid out in 256-byte steps.
struct Layout {
  int64_t total = 0;
  int64_t take(bool used, int64_t bytes) {
    if (!used) return -1;
    const int64_t r = total;
    total += align256(bytes);
    return r;
  }
};

// The forward's splits and scratch: copies of x and w, the splits' sums (byte offsets, -1: none).
struct FwdPlan {
  int split = 1;
  int64_t x = -1, w = -1, part = -1, total = 0;
};

// `any`: what any pointers and strides may need.
FwdPlan fwd_plan(const gs_linear_args* a, bool any) {
  FwdPlan p;
  if (a->dtype != GS_DTYPE_BF16 || gemm_bf16_few_rows((int)a->M, (int)a->N, (int)a->K)) return p;
  p.split = gemm_bf16_pick_split((int)a->M, (int)a->N, (int)a->K);
  Layout l;
  const bool pays = 2.0 * a->M * a->N * a->K >= kPadFlops;
  p.x = l.take(pays && (any || !granular(a->x, a->sx, a->K)), a->M * up8(a->K) * 2);
  p.w = l.take(pays && (any || !granular(a->w, a->K, a->K)), a->N * up8(a->K) * 2);
  p.part = l.take(p.split > 1, p.split * a->M * a->N * 4);
  p.total = l.total;
  return p;
}

// The backward's: dpre (rows of ldp), the column sums' parts, copies of x and w, the
// splits' sums of dx and of dw.
struct BwdPlan {
  int split_x, split_w;
  int64_t rows, ldp, dpre, cols, x, w, dx, dw, total;
};

BwdPlan bwd_plan(const gs_linear_bwd_args* a, bool any) {
  BwdPlan p{};
  const bool bf16 = a->dtype == GS_DTYPE_BF16, products = a->dx || a->dw;
  const int64_t size = bf16 ? 2 : 4;
  p.split_x = bf16 ? gemm_bf16_pick_split((int)a->M, (int)a->K, (int)a->N) : 1;
  p.split_w = bf16 ? gemm_bf16_pick_split((int)a->N, (int)a->K, (int)a->M) : gemm_pick_split((int)a->N, (int)a->K, (int)a->M);
  const bool pays = bf16 && 2.0 * a->M * a->N * a->K >= (a->dw ? kPadFlopsDw : kPadFlops);
  Layout l;
  p.ldp = pays ? up8(a->N) : a->N;
  p.dpre = l.take(products && (a->activation != GS_ACT_NONE || (pays && (any || !granular(a->dy, a->sdy, a->N)))),
                  a->M * p.ldp * size);
  p.rows = dpre_rows(a->M, a->N, bf16);
  p.cols = l.take(a->dbias != nullptr, (a->M + p.rows - 1) / p.rows * a->N * 4);
  p.x = l.take(pays && a->dw && (any || !granular(a->x, a->sx, a->K)), a->M * up8(a->K) * 2);
  p.w = l.take(pays && a->dx && (any || !granular(a->w, a->K, a->K)), a->N * up8(a->K) * 2);
  p.dx = l.take(a->dx && p.split_x > 1, p.split_x * a->M * a->K * 4);
  p.dw = l.take(a->dw && p.split_w > 1, p.split_w * a->N * a->K * 4);
  p.total = l.total;
  return p;
}

// Copies x [M, K] and w [N, K] (either may stay: offset -1) to rows of up8(K).
int pad(const void* x, int64_t sx, int64_t M, void* xp, const void* w, int64_t N, void* wp, int64_t K,
        hipStream_t stream) {
  if (xp == nullptr && wp == nullptr) return GS_OK;
  const int kp = (int)up8(K);
  PadJob a{static_cast<const __bf16*>(x), static_cast<__bf16*>(xp), sx, xp ? M * (kp / 8) : 0, (int)K, kp};
  PadJob b{static_cast<const __bf16*>(w), static_cast<__bf16*>(wp), K, wp ? N * (kp / 8) : 0, (int)K, kp};
  const int64_t groups = (a.octets + b.octets + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(pad_kernel, dim3((unsigned)std::min<int64_t>(groups, 8192)), dim3(kThreads), 0, stream, a, b);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int64_t gs_linear_scratch_bytes(const gs_linear_args* a) {
  clear_error();
  const int rc = check_fwd(a, "gs_linear_scratch_bytes");
  return rc ? rc : fwd_plan(a, !a->x || !a->w).total;
}

extern "C" int gs_linear_fwd(const gs_linear_args* a, hipStream_t stream) {
  const char* who = "gs_linear_fwd";
  clear_error();
  int rc = check_fwd(a, who);
  if (rc) return rc;
  if (!a->x || !a->w || !a->y) return set_error(GS_ERR_INVALID, "%s: x, w and y must be non-NULL device pointers", who);
  const FwdPlan plan = fwd_plan(a, false);
  if ((rc = check_scratch(who, a->scratch, a->scratch_bytes, plan.total))) return rc;
  char* scratch = static_cast<char*>(a->scratch);
  auto at = [&](int64_t off) -> void* { return off < 0 ? nullptr : scratch + off; };
  LinearEpilogue e;
  e.bias = a->bias;
  e.residual = a->residual;
  e.pre = a->pre;
  e.ldr = a->sr;
  e.act = a->activation;
  if (a->dtype == GS_DTYPE_BF16) {
    if ((rc = pad(a->x, a->sx, a->M, at(plan.x), a->w, a->N, at(plan.w), a->K, stream))) return rc;
    GemmBf16Args g;
    g.a = static_cast<const __bf16*>(plan.x < 0 ? a->x : at(plan.x));
    g.lda = plan.x < 0 ? a->sx : up8(a->K);
    g.b = static_cast<const __bf16*>(plan.w < 0 ? a->w : at(plan.w));
    g.ldb = plan.w < 0 ? a->K : up8(a->K);
    g.y = static_cast<__bf16*>(a->y);
    g.ldy = a->sy;
    g.part = static_cast<float*>(at(plan.part));
    g.epi = e;
    g.M = (int)a->M;
    g.N = (int)a->N;
    g.a_pads = plan.x >= 0;
    g.b_pads = plan.w >= 0;
    g.K = (int)a->K;
    g.ksplit = plan.split;
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
  g.has_epi = e.act != GS_ACT_NONE || e.residual != nullptr || e.pre != nullptr;
  g.epi = e;
  return gemm_f32(g, stream, who);
}

extern "C" int64_t gs_linear_bwd_scratch_bytes(const gs_linear_bwd_args* a) {
  clear_error();
  const int rc = check_bwd(a, "gs_linear_bwd_scratch_bytes");
  return rc ? rc : bwd_plan(a, !a->x || !a->w || !a->dy).total;
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
  const BwdPlan plan = bwd_plan(a, false);
  if ((rc = check_scratch(who, a->scratch, a->scratch_bytes, plan.total))) return rc;
  char* scratch = static_cast<char*>(a->scratch);
  auto at = [&](int64_t off) -> void* { return off < 0 ? nullptr : scratch + off; };
  const bool bf16 = a->dtype == GS_DTYPE_BF16;
  const int chunks = (int)((a->M + plan.rows - 1) / plan.rows);
  if (plan.dpre >= 0 || plan.cols >= 0) {
    DpreArgs p{act ? a->pre : nullptr, a->dy, at(plan.dpre), static_cast<float*>(at(plan.cols)), a->sdy, plan.ldp,
               (int)a->M, (int)a->N, a->activation, (int)plan.rows};
    for (int first = 0; first < chunks; first += 65535) {  // grid.y
      DpreArgs q = p;
      const int64_t r = (int64_t)first * plan.rows;
      const int64_t size = bf16 ? 2 : 4;
      q.M = (int)std::min<int64_t>(a->M - r, 65535 * plan.rows);
      if (q.pre) q.pre = static_cast<const char*>(q.pre) + r * a->N * size;
      q.dy = static_cast<const char*>(q.dy) + r * a->sdy * size;
      if (q.dpre) q.dpre = static_cast<char*>(q.dpre) + r * plan.ldp * size;
      if (q.part) q.part += (int64_t)first * a->N;
      auto fn = bf16 ? dpre_kernel<__bf16> : dpre_kernel<float>;
      const int cols = bf16 ? 128 : 64;
      hipLaunchKernelGGL(fn, dim3((unsigned)((a->N + cols - 1) / cols), (unsigned)((q.M + plan.rows - 1) / plan.rows)), dim3(kThreads),
                         0, stream, q);
      GS_CHECK_HIP(hipGetLastError());
    }
  }
  const void* dpre = plan.dpre >= 0 ? at(plan.dpre) : a->dy;
  const int64_t sd = plan.dpre >= 0 ? plan.ldp : a->sdy;
  const bool dpre_pads = plan.dpre >= 0 && plan.ldp == up8(a->N);
  if ((rc = pad(a->x, a->sx, a->M, at(plan.x), a->w, a->N, at(plan.w), a->K, stream))) return rc;
  ColumnSums sums;
  if (a->dbias != nullptr) {
    sums.dst = a->dbias;
    sums.src = static_cast<const float*>(at(plan.cols));
    sums.n = (int)a->N;
    sums.parts = chunks;
  }
  if (bf16) {
    GemmBf16Args x, w;
    x.a = w.a = static_cast<const __bf16*>(dpre);
    x.lda = w.lda = sd;
    x.a_pads = w.a_pads = dpre_pads;
    x.b = static_cast<const __bf16*>(plan.w < 0 ? a->w : at(plan.w));
    x.ldb = plan.w < 0 ? a->K : up8(a->K);
    x.b_pads = plan.w >= 0;
    x.y = static_cast<__bf16*>(a->dx);
    x.ldy = w.ldy = a->K;
    x.part = static_cast<float*>(at(plan.dx));
    x.M = (int)a->M;
    x.N = (int)a->K;
    x.K = (int)a->N;
    x.ksplit = plan.split_x;
    x.layout = kGemmNN;
    w.b = static_cast<const __bf16*>(plan.x < 0 ? a->x : at(plan.x));
    w.ldb = plan.x < 0 ? a->sx : up8(a->K);
    w.b_pads = plan.x >= 0;
    w.y = static_cast<__bf16*>(a->dw);
    w.part = static_cast<float*>(at(plan.dw));
    w.M = (int)a->N;
    w.N = (int)a->K;
    w.K = (int)a->M;
    w.ksplit = plan.split_w;
    w.layout = kGemmTN;
    if (a->dx && a->dw && gemm_bf16_pair_applies(x, w)) return gemm_bf16_pair(x, w, sums, stream, who);
    if (a->dx && (rc = gemm_bf16(x, stream, who))) return rc;
    if (a->dw && (rc = gemm_bf16(w, stream, who))) return rc;
  } else {
    GemmArgs x, w;
    x.a = w.a = static_cast<const float*>(dpre);
    x.lda = w.lda = sd;
    x.b = static_cast<const float*>(a->w);
    x.ldb = a->K;
    x.c = static_cast<float*>(a->dx);
    x.ldc = w.ldc = a->K;
    x.M = (int)a->M;
    x.N = (int)a->K;
    x.K = (int)a->N;
    x.layout = kGemmNN;
    w.b = static_cast<const float*>(a->x);
    w.ldb = a->sx;
    w.c = static_cast<float*>(plan.dw >= 0 ? at(plan.dw) : a->dw);
    w.split_stride = a->N * a->K;
    w.M = (int)a->N;
    w.N = (int)a->K;
    w.K = (int)a->M;
    w.ksplit = plan.split_w;
    w.layout = kGemmTN;
    if (a->dx && a->dw && gemm_pair_applies(x, w)) {
      if ((rc = gemm_pair(x, w, sums, stream, who))) return rc;
      sums.dst = nullptr;
    } else {
      if (a->dx && (rc = gemm_f32(x, stream, who))) return rc;
      if (a->dw && (rc = gemm_f32(w, stream, who))) return rc;
    }
    if (a->dw) {
      if (plan.dw >= 0 && (rc = sum_partials(static_cast<float*>(a->dw), w.c, a->N * a->K, plan.split_w, a->N * a->K, stream, who)))
        return rc;
    }
  }
  if (sums.dst != nullptr) {
    hipLaunchKernelGGL(bf16 ? sum_columns_kernel<__bf16> : sum_columns_kernel<float>, dim3((unsigned)((a->N + 15) / 16)),
                       dim3(kThreads), 0, stream, sums);
    GS_CHECK_HIP(hipGetLastError());
  }
  return GS_OK;
}
