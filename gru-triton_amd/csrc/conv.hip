// Short causal convolution of each channel over time (gfx950):
//   pre_t = bias + sum_k w[c][k] x_{t-W+1+k},  y = act(pre),  W = 2 to 4 taps,
// forward and backward, and one step of it for serving. Inputs before the first step are those of
// `state` (or zero); reset[t][b] != 0 starts a new sequence at step t, for which everything before
// counts as zero, whatever it holds.
//
// Backward, with g_t = dy_t act'(pre_t): dx_t = sum_j w[c][W-1-j] g_{t+j},
// dw[c][k] = sum_t g_t x_{t-W+1+k}, dbias = sum_t g_t, over the pairs of steps with no start between.
//
// Bound by memory. A lane holds V channels and walks a run of steps with the last W - 1 inputs (and, backwards, the
// W gradients that are not complete yet) in registers, so that each value is read once, but for the
// W - 1 at a run's ends. A backward workgroup's four waves take runs one after the other and join their sums over
// time, which a second launch adds up in order: results are reproducible. T 8192, B 8, C 2048, W 4 bf16: forward
// 113 us (4.7 TB/s), backward 197 (4.1 TB/s) and the second launch 5.
#include "gs_act.h"
#include "gs_seq.h"

namespace gs {
namespace {

constexpr int kMostTaps = 4;

struct ConvParams {
  const void *x, *w, *bias, *state;
  const uint8_t* reset;
  void *y, *last;                   // forward
  const void *dy, *dlast;           // backward only from here
  void *dx, *dstate;
  float* part;                      // [runs / 4][W + 1][C]
  int64_t sx_t, sx_b, sr_t, sr_b, sy_t, sy_b, sdy_t, sdy_b, sdx_t, sdx_b;
  int T, B, C;
  int blocks, runs, length;         // channel blocks, runs along the time axis and their steps
};

// V channels of a row in one access: V elements of T, aligned to their size together.
template <typename T, int V>
struct Vec {
  static constexpr int kWords = V * (int)sizeof(T) >= 4 ? V * (int)sizeof(T) / 4 : 1;
  typedef unsigned int u2v __attribute__((ext_vector_type(2)));
  typedef unsigned int u4v __attribute__((ext_vector_type(4)));
  struct Raw {
    unsigned int w[kWords];
  };
  static __device__ __forceinline__ Raw load(const void* base, uint32_t off) {
    Raw r;
    const auto b = bounded_rsrc(base, 0x7fffffffu);
    if constexpr (V == 1) {
      r.w[0] = Elem<T>::load(base, off);
    } else if constexpr (kWords == 2) {
      const auto x = __builtin_bit_cast(u2v, __builtin_amdgcn_raw_buffer_load_b64(b, (int)off, 0, 0));
      r.w[0] = x[0];
      r.w[1] = x[1];
    } else {
      const auto x = __builtin_bit_cast(u4v, __builtin_amdgcn_raw_buffer_load_b128(b, (int)off, 0, 0));
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[i] = x[i];
    }
    return r;
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&x)[V]) {
    if constexpr (V == 1) {
      x[0] = Elem<T>::value(r.w[0]);
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        x[2 * i] = __uint_as_float(r.w[i] << 16);
        x[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = __uint_as_float(r.w[i]);
    }
  }
  static __device__ __forceinline__ void store(void* base, uint32_t off, const float (&x)[V]) {
    const auto b = bounded_rsrc(base, 0x7fffffffu);
    if constexpr (V == 1) {
      Elem<T>::store(base, off, x[0]);
    } else if constexpr (sizeof(T) == 2) {
      typedef float f2v __attribute__((ext_vector_type(2)));
      typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
      static_assert(V == 4, "four bfloat16 a lane");
      const u2v q{__builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{x[0], x[1]}), bf2v)),
                  __builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{x[2], x[3]}), bf2v))};
      __builtin_amdgcn_raw_buffer_store_b64(q, b, (int)off, 0, 0);
    } else {
      static_assert(V == 4, "four floats a lane");
      const u4v q{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
      __builtin_amdgcn_raw_buffer_store_b128(q, b, (int)off, 0, 0);
    }
  }
};

// Where a wave is: 64 V channels of batch row b, steps t0 to t1.
template <int V>
struct Run {
  int b, run, t0, t1, ch, lane;
  bool ok, any;  // the lane's channels exist; the wave's run does
  __device__ __forceinline__ explicit Run(const ConvParams& p) {
    lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quads = (p.runs + 3) / 4;
    int g = blockIdx.x;
    const int block = g % p.blocks;
    g /= p.blocks;
    run = g % quads * 4 + wave;
    b = g / quads;
    any = run < p.runs;
    t0 = min(run * p.length, p.T);
    t1 = any ? min(p.T, t0 + p.length) : t0;
    ch = (block * 64 + lane) * V;
    ok = any && ch < p.C;
  }
};

template <typename T>
__device__ __forceinline__ const T* at_step(const void* base, int64_t st, int64_t sb, int t, int b) {
  return static_cast<const T*>(base) + t * st + b * sb;
}
// The input of step t >= 1 - W, and where it lies: before the first step in `state` [B][W - 1][C].
template <typename T, int V, int W>
__device__ __forceinline__ typename Vec<T, V>::Raw input(const ConvParams& p, int t, int b, uint32_t off, bool some = true) {
  if (t < 0) {
    if (p.state == nullptr || !some) return typename Vec<T, V>::Raw{};
    return Vec<T, V>::load(static_cast<const T*>(p.state) + ((int64_t)b * (W - 1) + t + W - 1) * p.C, off);
  }
  return Vec<T, V>::load(at_step<T>(p.x, p.sx_t, p.sx_b, t, b), some ? off : kOffNone);
}
__device__ __forceinline__ bool starts(const ConvParams& p, int t, int b) {
  return p.reset != nullptr && t >= 0 && t < p.T && p.reset[t * p.sr_t + b * p.sr_b] != 0;
}

template <typename T, int V, int W>
__device__ __forceinline__ void load_taps(const ConvParams& p, int ch, bool ok, float (&w)[W][V], float (&bias)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < W; ++k) w[k][v] = ok ? (float)static_cast<const T*>(p.w)[(int64_t)(ch + v) * W + k] : 0.0f;
    bias[v] = ok && p.bias != nullptr ? (float)static_cast<const T*>(p.bias)[ch + v] : 0.0f;
  }
}

// Flags of 32 steps from t as a mask (uniform).
__device__ __forceinline__ uint32_t start_mask(const ConvParams& p, int t, int b, int lane, int end) {
  if (p.reset == nullptr) return 0;
  bool f = false;
  if (lane < 32 && t + lane < end) f = p.reset[(t + lane) * p.sr_t + b * p.sr_b] != 0;
  return (uint32_t)__builtin_amdgcn_ballot_w64(f);
}

// The last W - 1 inputs before step t (past[W - 2] the newest), those before a start as zero.
template <typename T, int V, int W>
__device__ __forceinline__ void load_past(const ConvParams& p, int t, int b, uint32_t off, float (&past)[W - 1][V]) {
#pragma unroll
  for (int k = 0; k < W - 1; ++k) {
    const int s = t - (W - 1) + k;
    const bool start = starts(p, s, b);
    Vec<T, V>::unpack(input<T, V, W>(p, s, b, off, s >= 1 - W), past[k]);
    if (start) {
#pragma unroll
      for (int j = 0; j < k; ++j)
#pragma unroll
        for (int v = 0; v < V; ++v) past[j][v] = 0.0f;
    }
  }
}

constexpr int kAhead = 8;  // steps whose loads are in flight

template <typename T, int V, int W, bool SILU>
__global__ __launch_bounds__(256) void conv_fwd_kernel(ConvParams p) {
  typedef Vec<T, V> E;
  const Run<V> at(p);
  if (!at.any) return;  // uniform in the wave
  const uint32_t off = at.ok ? (uint32_t)(at.ch * (int)sizeof(T)) : kOffNone;
  float w[W][V], bias[V], past[W - 1][V];
  load_taps<T, V, W>(p, at.ch, at.ok, w, bias);
  typename E::Raw raw[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) raw[i] = E::load(at_step<T>(p.x, p.sx_t, p.sx_b, min(at.t0 + i, p.T - 1), at.b), at.t0 + i < at.t1 ? off : kOffNone);
  load_past<T, V, W>(p, at.t0, at.b, off, past);
  for (int t0 = at.t0; t0 < at.t1; t0 += kAhead) {
    const uint32_t mask = start_mask(p, t0, at.b, at.lane, at.t1);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int t = t0 + i;
      if (t >= at.t1) break;  // uniform
      float x[V], y[V];
      E::unpack(raw[i], x);
      const int next = t + kAhead;
      raw[i] = E::load(at_step<T>(p.x, p.sx_t, p.sx_b, min(next, p.T - 1), at.b), next < at.t1 ? off : kOffNone);
      if (mask >> i & 1) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
#pragma unroll
          for (int v = 0; v < V; ++v) past[k][v] = 0.0f;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        y[v] = bias[v];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) y[v] = __builtin_fmaf(w[k][v], past[k][v], y[v]);
        y[v] = __builtin_fmaf(w[W - 1][v], x[v], y[v]);
        if (SILU) y[v] = act_value<GS_ACT_SILU>(y[v]);
#pragma unroll
        for (int k = 0; k < W - 2; ++k) past[k][v] = past[k + 1][v];
        past[W - 2][v] = x[v];
      }
      E::store(const_cast<T*>(at_step<T>(p.y, p.sy_t, p.sy_b, t, at.b)), off, y);
    }
  }
  if (p.last != nullptr && at.run == p.runs - 1) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k) E::store(static_cast<T*>(p.last) + ((int64_t)at.b * (W - 1) + k) * p.C, off, past[k]);
  }
}

// A run goes on W - 1 steps past its end for the gradients that later steps send to its own;
// what those steps give the sums over time is the next run's.
template <typename T, int V, int W, bool SILU>
__global__ __launch_bounds__(256) void conv_bwd_kernel(ConvParams p) {
  typedef Vec<T, V> E;
  constexpr int kDeep = 4;
  __shared__ float red[4][W + 1][64 * V];
  const Run<V> at(p);
  const uint32_t off = at.ok ? (uint32_t)(at.ch * (int)sizeof(T)) : kOffNone;
  float w[W][V], bias[V], past[W - 1][V], acc[W][V], dw[W][V], db[V];
  load_taps<T, V, W>(p, at.ch, at.ok, w, bias);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    db[v] = 0.0f;
#pragma unroll
    for (int k = 0; k < W; ++k) acc[k][v] = dw[k][v] = 0.0f;
  }
  const int end = at.any ? min(p.T, at.t1 + W - 1) : at.t1;
  typename E::Raw rx[kDeep], rg[kDeep];
  auto fetch = [&](int i, int t) __attribute__((always_inline)) {
    const int r = min(t, p.T - 1);
    rx[i] = E::load(at_step<T>(p.x, p.sx_t, p.sx_b, r, at.b), t < end ? off : kOffNone);
    rg[i] = E::load(at_step<T>(p.dy, p.sdy_t, p.sdy_b, r, at.b), t < end ? off : kOffNone);
  };
#pragma unroll
  for (int i = 0; i < kDeep; ++i) fetch(i, at.t0 + i);
  int since = W;  // steps since the last start, W for all that is further back
  if (at.any) {
    load_past<T, V, W>(p, at.t0, at.b, off, past);
#pragma unroll
    for (int k = 1; k < W; ++k)
      if (starts(p, at.t0 - (W - k), at.b)) since = W - k - 1;
  }
  // dx of step t (also of the state's, t < 0) is complete
  auto put = [&](int t, float (&d)[V]) __attribute__((always_inline)) {
    if (t < 0) {
      if (p.dstate != nullptr) E::store(static_cast<T*>(p.dstate) + ((int64_t)at.b * (W - 1) + t + W - 1) * p.C, off, d);
    } else {
      E::store(const_cast<T*>(at_step<T>(p.dx, p.sdx_t, p.sdx_b, t, at.b)), off, d);
    }
  };
  const int first = at.run == 0 ? 1 - W : at.t0;  // the first step whose dx is this run's
  for (int t0 = at.t0; t0 < end; t0 += kDeep) {
    const uint32_t mask = start_mask(p, t0, at.b, at.lane, end);
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int t = t0 + i;
      if (t >= end) break;  // uniform
      float x[V], g[V], done[V];
      E::unpack(rx[i], x);
      E::unpack(rg[i], g);
      fetch(i, t + kDeep);
      since = mask >> i & 1 ? 0 : since + 1;
      if (since == 0) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
#pragma unroll
          for (int v = 0; v < V; ++v) past[k][v] = 0.0f;
      }
      const bool own = t < at.t1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (SILU) {
          float pre = bias[v];
#pragma unroll
          for (int k = 0; k < W - 1; ++k) pre = __builtin_fmaf(w[k][v], past[k][v], pre);
          pre = __builtin_fmaf(w[W - 1][v], x[v], pre);
          g[v] *= act_slope<GS_ACT_SILU>(pre);
        }
        if (own) {
#pragma unroll
          for (int k = 0; k < W - 1; ++k) dw[k][v] = __builtin_fmaf(g[v], past[k][v], dw[k][v]);
          dw[W - 1][v] = __builtin_fmaf(g[v], x[v], dw[W - 1][v]);
          db[v] += g[v];
        }
        // acc[k]: dx of step t - (W - 1) + k
#pragma unroll
        for (int k = 0; k < W; ++k)
          if (since >= W - 1 - k) acc[k][v] = __builtin_fmaf(w[k][v], g[v], acc[k][v]);
        done[v] = acc[0][v];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) acc[k][v] = acc[k + 1][v];
        acc[W - 1][v] = 0.0f;
#pragma unroll
        for (int k = 0; k < W - 2; ++k) past[k][v] = past[k + 1][v];
        past[W - 2][v] = x[v];
      }
      if (t - (W - 1) >= first) put(t - (W - 1), done);
    }
  }
  // the axis' last W - 1 steps (or, T being short, the state's), which `last` holds too
  if (at.any && end == p.T) {
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
      const int t = p.T - (W - 1) + k;
      if (t < first || t >= at.t1) continue;
      if (p.dlast != nullptr && since >= W - 2 - k) {
        float d[V];
        E::unpack(E::load(static_cast<const T*>(p.dlast) + ((int64_t)at.b * (W - 1) + k) * p.C, off), d);
#pragma unroll
        for (int v = 0; v < V; ++v) acc[k][v] += d[v];
      }
      put(t, acc[k]);
    }
  }
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < W; ++k) red[wave][k][at.lane * V + v] = dw[k][v];
    red[wave][W][at.lane * V + v] = db[v];
  }
  __syncthreads();
  const int block = blockIdx.x % p.blocks;
  for (int e = threadIdx.x; e < (W + 1) * 64 * V; e += 256) {
    const int k = e / (64 * V), c = e % (64 * V), ch = block * 64 * V + c;
    if (ch < p.C)
      p.part[((int64_t)(blockIdx.x / p.blocks) * (W + 1) + k) * p.C + ch] =
          ((red[0][k][c] + red[1][k][c]) + red[2][k][c]) + red[3][k][c];
  }
}

// dw [C][W] and dbias [C]: sums over the parts. Lanes are channels; a workgroup's sixteen waves
// take every sixteenth part, joined in order.
template <typename T>
__global__ __launch_bounds__(1024) void conv_sum_kernel(const float* part, void* dw, void* dbias, int C, int W, int parts) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ch = blockIdx.x * 64 + lane, k = blockIdx.y;
  const int64_t plane = (int64_t)(W + 1) * C;
  const float* src = part + (int64_t)k * C + ch;
  float s = 0.0f;
  if (ch < C) {
    for (int k0 = wave; k0 < parts; k0 += 16 * 8) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = k0 + 16 * i < parts ? src[(k0 + 16 * i) * plane] : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k0 + 16 * i < parts) s += x[i];
    }
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || ch >= C) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) s += red[w][lane];
  if (k < W && dw != nullptr) static_cast<T*>(dw)[(int64_t)ch * W + k] = (T)s;
  if (k == W && dbias != nullptr) static_cast<T*>(dbias)[ch] = (T)s;
}

// One token for each row of a batch of requests; rows of a cache [S][W - 1][C] hold their last
// inputs and move on by one. A lane a channel, one launch.
struct ConvStepParams {
  const void *x, *w, *bias;
  void* state;
  const int32_t* slots;
  void* y;
  int64_t sx, ss, sy;
  int B, C, S;
};

template <typename T, int W, bool SILU>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvStepParams p) {
  const int c = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
  if (c >= p.C) return;
  const int slot = p.slots ? p.slots[b] : b;
  T* out = static_cast<T*>(p.y) + b * p.sy + c;
  if (slot < 0 || slot >= p.S) {
    *out = (T)(slot < 0 ? 0.0f : __builtin_nanf(""));
    return;
  }
  const T* w = static_cast<const T*>(p.w) + (int64_t)c * W;
  T* s = static_cast<T*>(p.state) + slot * p.ss + c;
  T x[W];
#pragma unroll
  for (int k = 0; k < W - 1; ++k) x[k] = s[(int64_t)k * p.C];
  x[W - 1] = (static_cast<const T*>(p.x) + b * p.sx)[c];
  float y = p.bias ? (float)static_cast<const T*>(p.bias)[c] : 0.0f;
#pragma unroll
  for (int k = 0; k < W; ++k) y = __builtin_fmaf((float)w[k], (float)x[k], y);
#pragma unroll
  for (int k = 0; k < W - 1; ++k) s[(int64_t)k * p.C] = x[k + 1];
  *out = (T)(SILU ? act_value<GS_ACT_SILU>(y) : y);
}

// ---- host ---------------------------------------------------------------------------

struct Plan {
  int v, blocks, runs, length;
};

int64_t groups_of(const Plan& p, int64_t B) { return (int64_t)p.blocks * ((p.runs + 3) / 4) * B; }

// Runs of 128 steps at most, whose ends cost little, and shorter ones, of 8 at least, where there are fewer than a
// thousand waves (T 2000, B 16, C 96: 38 us with four thousand asked for, 35 with one).
Plan make_plan(int64_t T, int64_t B, int64_t C, int v) {
  Plan r;
  r.v = v;
  r.blocks = (int)((C + 64 * v - 1) / (64 * v));
  const int64_t steps = r.blocks * B * T;
  int64_t length = 128;
  while (length > 8 && steps / length < 1024) length /= 2;
  r.length = (int)length;
  r.runs = (int)((T + length - 1) / length);
  return r;
}

struct Strided {
  const void* p;
  int64_t st, sb;
};
// Four channels a lane where every row allows the access and there are lanes enough for them (a training step of
// T 8192, B 8, C 2048 bf16 takes 322 us so and 521 with one; T 2000, B 16, C 96: 50 and 55).
Plan plan_of(int dtype, int64_t T, int64_t B, int64_t C, const Strided* t, int count) {
  const int bytes = dtype == GS_DTYPE_F32 ? 16 : 8;
  bool four = C % 4 == 0 && C >= 64;
  for (int i = 0; i < count; ++i)
    four = four && (reinterpret_cast<uintptr_t>(t[i].p) & (uintptr_t)(bytes - 1)) == 0 && t[i].st % 4 == 0 && t[i].sb % 4 == 0;
  return make_plan(T, B, C, four ? 4 : 1);
}

typedef void (*ConvFn)(ConvParams);
template <typename T, int V, int W>
ConvFn kernel_in(bool back, bool silu) {
  if (back) return silu ? conv_bwd_kernel<T, V, W, true> : conv_bwd_kernel<T, V, W, false>;
  return silu ? conv_fwd_kernel<T, V, W, true> : conv_fwd_kernel<T, V, W, false>;
}
template <typename T, int V>
ConvFn kernel_for(int W, bool back, bool silu) {
  return W == 2 ? kernel_in<T, V, 2>(back, silu) : W == 3 ? kernel_in<T, V, 3>(back, silu) : kernel_in<T, V, 4>(back, silu);
}
ConvFn kernel_of(int dtype, int v, int W, bool back, bool silu) {
  if (dtype == GS_DTYPE_F32) return v == 4 ? kernel_for<float, 4>(W, back, silu) : kernel_for<float, 1>(W, back, silu);
  return v == 4 ? kernel_for<__bf16, 4>(W, back, silu) : kernel_for<__bf16, 1>(W, back, silu);
}

int check_sizes(const char* who, int64_t T, int64_t B, int64_t C, int64_t W, int dtype, int activation) {
  if (T < 1) return set_error(GS_ERR_INVALID, "%s: seq length T must be > 0; got T=%lld", who, (long long)T);
  if (B < 1) return set_error(GS_ERR_INVALID, "%s: batch size B must be > 0; got B=%lld", who, (long long)B);
  if (C < 1) return set_error(GS_ERR_INVALID, "%s: channels C must be > 0; got C=%lld", who, (long long)C);
  if (W < 2 || W > kMostTaps)
    return set_error(GS_ERR_INVALID, "%s: taps W must be 2 to %d; got W=%lld", who, kMostTaps, (long long)W);
  if (T > (1ll << 30) || B > (1ll << 20) || C > (1ll << 20))
    return set_error(GS_ERR_INVALID, "%s: T/B/C out of supported range (T=%lld, B=%lld, C=%lld)", who, (long long)T,
                     (long long)B, (long long)C);
  if (activation != GS_ACT_NONE && activation != GS_ACT_SILU)
    return set_error(GS_ERR_INVALID, "%s: activation must be none or silu; got %d", who, activation);
  return check_dtype(who, dtype);
}

int check_fwd(const gs_conv_args* a, const char* who) {
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  int rc = check_sizes(who, a->T, a->B, a->C, a->W, a->dtype, a->activation);
  if (rc) return rc;
  if ((rc = check_step_rows(who, "x", a->T, a->B, a->C, a->sx_t, a->sx_b, false))) return rc;
  if ((rc = check_step_rows(who, "reset", a->T, a->B, 1, a->sr_t, a->sr_b, false))) return rc;
  return check_step_rows(who, "y", a->T, a->B, a->C, a->sy_t, a->sy_b, true);
}
int check_bwd(const gs_conv_bwd_args* a, const char* who) {
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  int rc = check_sizes(who, a->T, a->B, a->C, a->W, a->dtype, a->activation);
  if (rc) return rc;
  if ((rc = check_step_rows(who, "x", a->T, a->B, a->C, a->sx_t, a->sx_b, false))) return rc;
  if ((rc = check_step_rows(who, "reset", a->T, a->B, 1, a->sr_t, a->sr_b, false))) return rc;
  if ((rc = check_step_rows(who, "dy", a->T, a->B, a->C, a->sdy_t, a->sdy_b, false))) return rc;
  return check_step_rows(who, "dx", a->T, a->B, a->C, a->sdx_t, a->sdx_b, true);
}

Plan plan_fwd(const gs_conv_args* a) {
  const Strided t[4] = {{a->x, a->sx_t, a->sx_b}, {a->y, a->sy_t, a->sy_b}, {a->state, 0, 0}, {a->last, 0, 0}};
  return plan_of(a->dtype, a->T, a->B, a->C, t, 4);
}
Plan plan_bwd(const gs_conv_bwd_args* a) {
  const Strided t[6] = {{a->x, a->sx_t, a->sx_b}, {a->dy, a->sdy_t, a->sdy_b}, {a->dx, a->sdx_t, a->sdx_b},
                        {a->state, 0, 0}, {a->dstate, 0, 0}, {a->dlast, 0, 0}};
  return plan_of(a->dtype, a->T, a->B, a->C, t, 6);
}
int64_t part_bytes(const Plan& p, int64_t B, int64_t C, int64_t W) { return align256((p.runs + 3) / 4 * B * (W + 1) * C * 4); }

template <typename Args>
ConvParams params_of(const Args* a, const Plan& plan) {
  ConvParams p{};
  p.x = a->x;
  p.w = a->w;
  p.bias = a->bias;
  p.state = a->state;
  p.reset = a->reset;
  p.sx_t = a->sx_t;
  p.sx_b = a->sx_b;
  p.sr_t = a->sr_t;
  p.sr_b = a->sr_b;
  p.T = (int)a->T;
  p.B = (int)a->B;
  p.C = (int)a->C;
  p.blocks = plan.blocks;
  p.runs = plan.runs;
  p.length = plan.length;
  return p;
}

int fits_launch(const char* who, const Plan& plan, int64_t T, int64_t B, int64_t C) {
  if (groups_of(plan, B) * 256 > UINT32_MAX)
    return set_error(GS_ERR_INVALID, "%s: more workgroups than a launch holds (T=%lld, B=%lld, C=%lld)", who, (long long)T,
                     (long long)B, (long long)C);
  return GS_OK;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_conv_fwd(const gs_conv_args* a, hipStream_t stream) {
  const char* who = "gs_conv_fwd";
  clear_error();
  int rc = check_fwd(a, who);
  if (rc) return rc;
  if (!a->x || !a->w || !a->y) return set_error(GS_ERR_INVALID, "%s: x, w and y must be non-NULL device pointers", who);
  const Plan plan = plan_fwd(a);
  if ((rc = fits_launch(who, plan, a->T, a->B, a->C))) return rc;
  ConvParams p = params_of(a, plan);
  p.y = a->y;
  p.last = a->last;
  p.sy_t = a->sy_t;
  p.sy_b = a->sy_b;
  hipLaunchKernelGGL(kernel_of(a->dtype, plan.v, (int)a->W, false, a->activation == GS_ACT_SILU),
                     dim3((unsigned)groups_of(plan, a->B)), dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}

extern "C" int64_t gs_conv_bwd_scratch_bytes(const gs_conv_bwd_args* a) {
  clear_error();
  const int rc = check_bwd(a, "gs_conv_bwd_scratch_bytes");
  if (rc) return rc;
  return std::max(part_bytes(make_plan(a->T, a->B, a->C, 1), a->B, a->C, a->W),
                  part_bytes(make_plan(a->T, a->B, a->C, 4), a->B, a->C, a->W));
}

extern "C" int gs_conv_bwd(const gs_conv_bwd_args* a, hipStream_t stream) {
  const char* who = "gs_conv_bwd";
  clear_error();
  int rc = check_bwd(a, who);
  if (rc) return rc;
  if (!a->x || !a->w || !a->dy || !a->dx)
    return set_error(GS_ERR_INVALID, "%s: x, w, dy and dx must be non-NULL device pointers", who);
  const Plan plan = plan_bwd(a);
  if ((rc = fits_launch(who, plan, a->T, a->B, a->C))) return rc;
  if ((rc = check_plain_scratch(who, a->scratch, a->scratch_bytes, part_bytes(plan, a->B, a->C, a->W)))) return rc;
  ConvParams p = params_of(a, plan);
  p.dy = a->dy;
  p.dlast = a->dlast;
  p.dx = a->dx;
  p.dstate = a->dstate;
  p.part = static_cast<float*>(a->scratch);
  p.sdy_t = a->sdy_t;
  p.sdy_b = a->sdy_b;
  p.sdx_t = a->sdx_t;
  p.sdx_b = a->sdx_b;
  hipLaunchKernelGGL(kernel_of(a->dtype, plan.v, (int)a->W, true, a->activation == GS_ACT_SILU),
                     dim3((unsigned)groups_of(plan, a->B)), dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  if (a->dw != nullptr || a->dbias != nullptr) {
    hipLaunchKernelGGL(a->dtype == GS_DTYPE_F32 ? conv_sum_kernel<float> : conv_sum_kernel<__bf16>,
                       dim3((unsigned)((a->C + 63) / 64), (unsigned)(a->W + 1)), dim3(1024), 0, stream, p.part, a->dw, a->dbias,
                       (int)a->C, (int)a->W, (int)((plan.runs + 3) / 4 * a->B));
    GS_CHECK_HIP(hipGetLastError());
  }
  return GS_OK;
}

extern "C" int gs_conv_step(const gs_conv_step_args* a, hipStream_t stream) {
  const char* who = "gs_conv_step";
  clear_error();
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  const int rc = check_sizes(who, 1, a->B, a->C, a->W, a->dtype, a->activation);
  if (rc) return rc;
  if (!a->x || !a->w || !a->state || !a->y)
    return set_error(GS_ERR_INVALID, "%s: x, w, state and y must be non-NULL device pointers", who);
  if (a->S < 1 || a->S > (1ll << 30) || (a->slots == nullptr && a->S < a->B))
    return set_error(GS_ERR_INVALID, "%s: a cache of S=%lld states does not hold B=%lld rows", who, (long long)a->S,
                     (long long)a->B);
  if (a->sx < 0 || (a->S > 1 && a->ss < (a->W - 1) * a->C) || (a->B > 1 && a->sy < a->C))
    return set_error(GS_ERR_INVALID, "%s: strides (x %lld, state %lld, y %lld) do not describe rows of C=%lld", who,
                     (long long)a->sx, (long long)a->ss, (long long)a->sy, (long long)a->C);
  if (a->B > 65535) return set_error(GS_ERR_INVALID, "%s: B=%lld exceeds 65535", who, (long long)a->B);
  ConvStepParams p{a->x, a->w, a->bias, a->state, a->slots, a->y, a->sx, a->ss, a->sy, (int)a->B, (int)a->C, (int)a->S};
  const bool silu = a->activation == GS_ACT_SILU;
  void (*fn)(ConvStepParams);
  if (a->dtype == GS_DTYPE_F32)
    fn = a->W == 2 ? (silu ? conv_step_kernel<float, 2, true> : conv_step_kernel<float, 2, false>)
       : a->W == 3 ? (silu ? conv_step_kernel<float, 3, true> : conv_step_kernel<float, 3, false>)
                   : (silu ? conv_step_kernel<float, 4, true> : conv_step_kernel<float, 4, false>);
  else
    fn = a->W == 2 ? (silu ? conv_step_kernel<__bf16, 2, true> : conv_step_kernel<__bf16, 2, false>)
       : a->W == 3 ? (silu ? conv_step_kernel<__bf16, 3, true> : conv_step_kernel<__bf16, 3, false>)
                   : (silu ? conv_step_kernel<__bf16, 4, true> : conv_step_kernel<__bf16, 4, false>);
  hipLaunchKernelGGL(fn, dim3((unsigned)((a->C + 255) / 256), (unsigned)a->B), dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}
