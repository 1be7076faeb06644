// Gated linear recurrence (gfx950): the GRU update without its hidden map,
//   z = sigmoid(gi_z), n = tanh(gi_n) or gi_n, h_t = z h_{t-1} + (1 - z) n,
// over T steps of B H independent channels, forward and backward, and one step of
// it for serving. reset[t][b] != 0 starts a new sequence at step t: h_{t-1} is
// taken as 0 there, whatever it holds (NaN and infinity included).
//
// With a_t = z (or "drop the carry") and b_t = (1 - z) n a step is the map
// h -> a h + b, and maps compose: (a2, b2) after (a1, b1) is (a2 a1, a2 b1 + b2).
// The backward is the same scan the other way: with D_t the gradient of h_t,
// E_t = a_t D_t the gradient it sends to h_{t-1} and d_t = dout[t],
//   D_t = d_t + E_{t+1},  E_t = a_t D_t  (E_T = dh_last, dh0 = E_0),
//   dgi_z = D (h_{t-1} - n) z (1 - z),  dgi_n = D (1 - z) (1 - n^2 if tanh).
//
// Layout: a workgroup owns LC V channels of one batch row and walks the time
// axis in tiles of 64 / LC x NW x U steps. A lane holds U consecutive steps of V
// channels in registers: it folds them to one map, the maps are scanned across
// the wave's 64 / LC step groups and, through LDS, its NW waves, and the lane
// then runs its U steps from its own carry. Each input is read once, the state
// between tiles stays in registers, and the next tile's loads are in flight
// meanwhile. Sums and states are fp32; the order of every operation is fixed by
// the sizes, so results are reproducible.
#include "gs_mfma.h"

namespace gs {
namespace {

typedef unsigned int u2v __attribute__((ext_vector_type(2)));
typedef unsigned int u4v __attribute__((ext_vector_type(4)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));

struct GlrParams {
  const void* gi;
  const float* h0;
  const uint8_t* reset;
  void* out;           // forward: written; backward: read
  float* h_last;
  const void* dout;    // backward only from here
  const float* dh_last;
  void* dgi;
  float* dh0;
  f2v* agg;            // [segments - 1][B][H] maps of whole segments, or NULL
  int64_t sg_t, sg_b, sh0_b, sr_t, sr_b, so_t, so_b, sd_t, sd_b, sdg_t, sdg_b;
  int T, B, H;
  int blocks;          // channel blocks per batch row
  int seg;             // steps per segment (a multiple of the tile)
};

// The map h -> a h + b. A reset is a = -0 (a is never negative otherwise; a NaN
// of either sign comes with b = NaN): the carry is then dropped, not multiplied.
struct Map {
  float a, b;
};
template <bool RESET>
__device__ __forceinline__ float apply(const Map& m, float h) {
  const float x = __builtin_fmaf(m.a, h, m.b);
  return RESET && (int)__float_as_uint(m.a) < 0 ? m.b : x;
}
template <bool RESET>
__device__ __forceinline__ Map then(const Map& first, const Map& second) {
  Map r{second.a * first.a, __builtin_fmaf(second.a, first.b, second.b)};
  if (RESET && (int)__float_as_uint(second.a) < 0) r = second;
  return r;
}

// V elements of type T in one buffer access.
template <typename T, int V>
struct Pack {
  static constexpr int kBytes = V * (int)sizeof(T);
  static_assert(kBytes == 2 || kBytes == 4 || kBytes == 8, "2, 4 or 8 bytes a lane");
  typedef typename std::conditional<kBytes == 8, u2v, unsigned int>::type Raw;
  static __device__ __forceinline__ Raw load(const void* base, uint32_t off) {
    const auto r = bounded_rsrc(base, 0x7fffffffu);
    if constexpr (kBytes == 2)
      return (unsigned int)(unsigned short)__builtin_amdgcn_raw_buffer_load_b16(r, (int)off, 0, 0);
    else if constexpr (kBytes == 4)
      return __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0);
    else
      return __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0);
  }
  static __device__ __forceinline__ void store(void* base, uint32_t off, const float (&x)[V]) {
    const auto r = bounded_rsrc(base, 0x7fffffffu);
    if constexpr (sizeof(T) == 4) {
      if constexpr (V == 1)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[0]), r, (int)off, 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b64(u2v{__float_as_uint(x[0]), __float_as_uint(x[1])}, r, (int)off, 0, 0);
    } else if constexpr (V == 1) {
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (__bf16)x[0]), r, (int)off, 0, 0);
    } else {
      unsigned int w[V / 2];
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        w[i] = __builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{x[2 * i], x[2 * i + 1]}), bf2v));
      if constexpr (V == 2)
        __builtin_amdgcn_raw_buffer_store_b32(w[0], r, (int)off, 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b64(u2v{w[0], w[1]}, r, (int)off, 0, 0);
    }
  }
  static __device__ __forceinline__ void unpack(const Raw& w, float (&x)[V]) {
    if constexpr (sizeof(T) == 4) {
      if constexpr (V == 1)
        x[0] = __uint_as_float(w);
      else {
        x[0] = __uint_as_float(w[0]);
        x[1] = __uint_as_float(w[1]);
      }
    } else if constexpr (V == 1) {
      x[0] = __uint_as_float(w << 16);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        unsigned int u;
        if constexpr (V == 2)
          u = w;
        else
          u = w[i];
        x[2 * i] = __uint_as_float(u << 16);
        x[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
      }
    }
  }
};

template <bool TANH>
__device__ __forceinline__ void gates(float gz, float gn, float& z, float& n) {
  z = sigmoid(gz);
  n = TANH ? tanh_near(gn) : gn;
}

// Where a lane is: its channels, its step group, and its wave (uniform).
template <int V, int LC, int NW>
struct Place {
  static constexpr int NG = 64 / LC;
  int b, j, lc, lg, wave;
  bool ok, any;  // the lane's channels exist; the workgroup's do
  __device__ __forceinline__ Place(const GlrParams& p) {
    const int lane = threadIdx.x & 63;
    wave = NW > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    lc = lane % LC;
    lg = lane / LC;
    // neighbours in a row, which share cache lines, on one XCD (workgroup mod 8)
    const int per = gridDim.x >> 3, group = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    b = group / p.blocks;
    any = b < p.B;
    j = ((group - b * p.blocks) * LC + lc) * V;
    ok = any && j < p.H;
  }
};

// The maps before a lane's own steps: given each lane's map of its U steps,
// returns the state at the lane's first step and advances `carry` past the tile.
// `lds` is one of two buffers used in turn: a wave writes a buffer again only
// after a barrier that every wave reaches when it has read it.
template <int V, int LC, int NW, bool RESET>
__device__ __forceinline__ void enter(const Place<V, LC, NW>& at, Map (&m)[V], float (&carry)[V], float (&h)[V],
                                      Map (*lds)[LC * V]) {
  constexpr int NG = 64 / LC;
  Map before[V];
  if constexpr (NG > 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int d = 1; d < NG; d *= 2) {
        const Map o{__shfl_up(m[v].a, d * LC), __shfl_up(m[v].b, d * LC)};
        if (at.lg >= d) m[v] = then<RESET>(o, m[v]);
      }
      before[v] = Map{__shfl_up(m[v].a, LC), __shfl_up(m[v].b, LC)};
      if (at.lg == 0) before[v] = Map{1.0f, 0.0f};
    }
  }
  if constexpr (NW == 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = NG > 1 ? apply<RESET>(before[v], carry[v]) : carry[v];
      Map whole = m[v];
      if constexpr (NG > 1) whole = Map{__shfl(m[v].a, 64 - LC + at.lc), __shfl(m[v].b, 64 - LC + at.lc)};
      carry[v] = apply<RESET>(whole, carry[v]);
    }
  } else {
    if (at.lg == NG - 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) lds[at.wave][at.lc * V + v] = m[v];
    }
    lds_barrier();
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float c = carry[v], mine = c;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        if (w == at.wave) mine = c;
        c = apply<RESET>(lds[w][at.lc * V + v], c);
      }
      carry[v] = c;
      h[v] = NG > 1 ? apply<RESET>(before[v], mine) : mine;
    }
  }
}

// The state with which a segment starts: the first one's, taken through the maps
// of the segments before it.
template <int V, bool RESET>
__device__ __forceinline__ void segment_carry(const GlrParams& p, const float* first, int64_t ld, int b, int j, bool ok,
                                              float (&carry)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float c = first != nullptr && ok ? first[(int64_t)b * ld + j + v] : 0.0f;
    const f2v* a = p.agg + (int64_t)b * p.H + j + v;
    for (int s = 0; s < (int)blockIdx.y; ++s) {
      const f2v x = ok ? a[(int64_t)s * p.B * p.H] : f2v{1.0f, 0.0f};
      c = apply<RESET>(Map{x[0], x[1]}, c);
    }
    carry[v] = c;
  }
}

// Loads of U steps. Step i of a lane is t0 + lg U + i forwards, and t0 - lg U - i
// backwards (BACK); rem is how many of its steps exist. Offsets are the lane's
// part only (its channel and its group's distance from the wave's base); the
// base moves with i and the wave, in scalar registers.
template <typename T, int V, int U, bool BACK, bool FULL>
__device__ __forceinline__ void load_steps(const void* base, int64_t st, uint32_t off, int rem,
                                           typename Pack<T, V>::Raw (&x)[U]) {
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const T* q = static_cast<const T*>(base) + (BACK ? -i : i) * st;
    x[i] = Pack<T, V>::load(q, FULL || i < rem ? off : kOffNone);
  }
}

template <typename T, int V, int LC, int NW, int U, bool TANH, bool RESET>
__global__ __launch_bounds__(64 * NW) void glr_fwd_kernel(GlrParams p) {
  typedef Pack<T, V> P;
  constexpr int NG = 64 / LC, kTile = NG * NW * U;
  __shared__ Map lds[2][NW > 1 ? NW : 1][LC * V];
  const Place<V, LC, NW> at(p);
  if (!at.any) return;  // uniform
  const int tbeg = blockIdx.y * p.seg, tend = min(p.T, tbeg + p.seg);
  float carry[V];
  segment_carry<V, RESET>(p, p.h0, p.sh0_b, at.b, at.j, at.ok, carry);

  const T* gi = static_cast<const T*>(p.gi) + at.b * p.sg_b;
  T* out = static_cast<T*>(p.out) + at.b * p.so_b;
  const uint8_t* rs = RESET ? p.reset + at.b * p.sr_b : nullptr;
  const uint32_t lane_g = (uint32_t)((at.lg * U * p.sg_t + at.j) * sizeof(T));
  const uint32_t off_z = at.ok ? lane_g : kOffNone;
  const uint32_t off_n = at.ok ? lane_g + (uint32_t)(p.H * sizeof(T)) : kOffNone;
  const uint32_t off_o = at.ok ? (uint32_t)((at.lg * U * p.so_t + at.j) * sizeof(T)) : kOffNone;
  struct Set {
    typename P::Raw z[U], n[U];
    unsigned int r[U];
  };
  auto load = [&](int t0, Set& s) __attribute__((always_inline)) {
    const int tw = t0 + at.wave * NG * U;  // the wave's first step
    const T* g = gi + tw * p.sg_t;
    const int rem = tend - tw - at.lg * U;
    load_steps<T, V, U, false, false>(g, p.sg_t, off_z, rem, s.z);
    load_steps<T, V, U, false, false>(g, p.sg_t, off_n, rem, s.n);
    if constexpr (RESET) {
#pragma unroll
      for (int i = 0; i < U; ++i) s.r[i] = i < rem ? rs[(tw + at.lg * U + i) * p.sr_t] : 0u;
    }
  };
  auto tile = [&](int t0, const Set& s, Map (*buf)[LC * V]) __attribute__((always_inline)) {
    const int tw = t0 + at.wave * NG * U;
    const int rem = tend - tw - at.lg * U;
    Map m[V], e[U][V];
#pragma unroll
    for (int v = 0; v < V; ++v) m[v] = Map{1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float gz[V], gn[V];
      P::unpack(s.z[i], gz);
      P::unpack(s.n[i], gn);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float z, n;
        gates<TANH>(gz[v], gn[v], z, n);
        e[i][v] = Map{z, __builtin_fmaf(-z, n, n)};
        if (RESET && s.r[i]) e[i][v].a = -0.0f;
        if (i >= rem) e[i][v] = Map{1.0f, 0.0f};
        m[v] = then<RESET>(m[v], e[i][v]);
      }
    }
    float h[V];
    enter<V, LC, NW, RESET>(at, m, carry, h, buf);
    T* o = out + tw * p.so_t;
#pragma unroll
    for (int i = 0; i < U; ++i) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = apply<RESET>(e[i][v], h[v]);
      P::store(o + i * p.so_t, i < rem ? off_o : kOffNone, h);
    }
  };
  Set s0, s1;
  load(tbeg, s0);
  for (int t0 = tbeg; t0 < tend; t0 += 2 * kTile) {  // tend - tbeg >= 1
    load(t0 + kTile, s1);
    tile(t0, s0, lds[0]);
    if (t0 + kTile >= tend) break;
    load(t0 + 2 * kTile, s0);
    tile(t0 + kTile, s1, lds[1]);
  }
  if (p.h_last != nullptr && tend == p.T && at.ok && at.lg == 0 && at.wave == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) p.h_last[(int64_t)at.b * p.H + at.j + v] = carry[v];
  }
}

// The same walk from the last step to the first: tau = T - 1 - t counts up.
template <typename T, int V, int LC, int NW, int U, bool TANH, bool RESET>
__global__ __launch_bounds__(64 * NW) void glr_bwd_kernel(GlrParams p) {
  typedef Pack<T, V> P;
  constexpr int NG = 64 / LC, kTile = NG * NW * U;
  __shared__ Map lds[2][NW > 1 ? NW : 1][LC * V];
  const Place<V, LC, NW> at(p);
  if (!at.any) return;  // uniform
  const int tbeg = blockIdx.y * p.seg, tend = min(p.T, tbeg + p.seg);  // in tau
  float carry[V];
  segment_carry<V, RESET>(p, p.dh_last, p.H, at.b, at.j, at.ok, carry);

  const T* gi = static_cast<const T*>(p.gi) + at.b * p.sg_b;
  const T* out = static_cast<const T*>(p.out) + at.b * p.so_b;
  const T* dout = static_cast<const T*>(p.dout) + at.b * p.sd_b;
  T* dgi = static_cast<T*>(p.dgi) + at.b * p.sdg_b;
  const uint8_t* rs = RESET ? p.reset + at.b * p.sr_b : nullptr;
  // the wave's base is its last group's first step, the earliest in time
  const int back = (NG - 1 - at.lg) * U;
  auto lane_off = [&](int64_t st) { return (uint32_t)((back * st + at.j) * sizeof(T)); };
  const uint32_t off_h = (uint32_t)(p.H * sizeof(T));
  const uint32_t off_z = at.ok ? lane_off(p.sg_t) : kOffNone, off_n = at.ok ? off_z + off_h : kOffNone;
  const uint32_t off_o = at.ok ? lane_off(p.so_t) : kOffNone, off_d = at.ok ? lane_off(p.sd_t) : kOffNone;
  const uint32_t off_dz = at.ok ? lane_off(p.sdg_t) : kOffNone, off_dn = at.ok ? off_dz + off_h : kOffNone;
  struct Set {
    typename P::Raw z[U], n[U], h[U], d[U];
    unsigned int r[U];
  };
  auto load = [&](int t0, Set& s) __attribute__((always_inline)) {
    const int tw = t0 + at.wave * NG * U;  // the wave's first tau
    const int64_t t = p.T - 1 - tw - (NG - 1) * U;
    const int rem = tend - tw - at.lg * U;
    const int before = p.T - 1 - tw - at.lg * U;  // steps before the lane's first: step i has h_{t-1} in `out` if i < before
    load_steps<T, V, U, true, false>(gi + t * p.sg_t, p.sg_t, off_z, rem, s.z);
    load_steps<T, V, U, true, false>(gi + t * p.sg_t, p.sg_t, off_n, rem, s.n);
    load_steps<T, V, U, true, false>(dout + t * p.sd_t, p.sd_t, off_d, rem, s.d);
    load_steps<T, V, U, true, false>(out + (t - 1) * p.so_t, p.so_t, off_o, min(rem, before), s.h);
    if constexpr (RESET) {
#pragma unroll
      for (int i = 0; i < U; ++i) s.r[i] = i < rem ? rs[(int64_t)(before - i) * p.sr_t] : 0u;
    }
  };
  auto tile = [&](int t0, const Set& s, Map (*buf)[LC * V]) __attribute__((always_inline)) {
    const int tw = t0 + at.wave * NG * U;
    const int rem = tend - tw - at.lg * U;
    const int before = p.T - 1 - tw - at.lg * U;
    Map m[V];
    float z[U][V], n[U][V], d[U][V], hp[U][V];
#pragma unroll
    for (int v = 0; v < V; ++v) m[v] = Map{1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float gz[V], gn[V];
      P::unpack(s.z[i], gz);
      P::unpack(s.n[i], gn);
      P::unpack(s.d[i], d[i]);
      P::unpack(s.h[i], hp[i]);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        gates<TANH>(gz[v], gn[v], z[i][v], n[i][v]);
        Map e{z[i][v], z[i][v] * d[i][v]};
        if (RESET && s.r[i]) e = Map{-0.0f, 0.0f};
        if (i >= rem) e = Map{1.0f, 0.0f};
        m[v] = then<RESET>(m[v], e);
      }
    }
    // step 0 continues h0
    if (before < U && before >= 0 && rem > before && at.ok) {
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (i == before) {
#pragma unroll
          for (int v = 0; v < V; ++v) hp[i][v] = p.h0 ? p.h0[at.b * p.sh0_b + at.j + v] : 0.0f;
        }
    }
    float E[V];
    enter<V, LC, NW, RESET>(at, m, carry, E, buf);
    const int64_t t = p.T - 1 - tw - (NG - 1) * U;
    T* o = dgi + t * p.sdg_t;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float dz[V], dn[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float D = d[i][v] + E[v], a = z[i][v], c = n[i][v];
        const float h = RESET && s.r[i] ? 0.0f : hp[i][v];
        const float keep = D * (1.0f - a);
        dz[v] = keep * a * (h - c);
        dn[v] = TANH ? keep * __builtin_fmaf(-c, c, 1.0f) : keep;
        E[v] = RESET && s.r[i] ? 0.0f : a * D;
      }
      P::store(o - i * p.sdg_t, i < rem ? off_dz : kOffNone, dz);
      P::store(o - i * p.sdg_t, i < rem ? off_dn : kOffNone, dn);
    }
  };
  Set s0, s1;
  load(tbeg, s0);
  for (int t0 = tbeg; t0 < tend; t0 += 2 * kTile) {
    load(t0 + kTile, s1);
    tile(t0, s0, lds[0]);
    if (t0 + kTile >= tend) break;
    load(t0 + 2 * kTile, s0);
    tile(t0 + kTile, s1, lds[1]);
  }
  if (p.dh0 != nullptr && tend == p.T && at.ok && at.lg == 0 && at.wave == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) p.dh0[(int64_t)at.b * p.H + at.j + v] = carry[v];
  }
}

// The map of a whole segment, for axes so long that they are walked in several
// segments at once: each step group folds its own share of the segment's steps,
// then the shares are joined in order. The last segment's map is not needed.
template <typename T, int V, int LC, int NW, int U, bool TANH, bool RESET, bool BACK>
__global__ __launch_bounds__(64 * NW) void glr_segment_kernel(GlrParams p) {
  typedef Pack<T, V> P;
  constexpr int NG = 64 / LC;
  __shared__ Map lds[NW][LC * V];
  const Place<V, LC, NW> at(p);
  if (!at.any) return;  // uniform
  const int tbeg = blockIdx.y * p.seg, share = p.seg / (NG * NW);  // a multiple of U
  const int first = tbeg + (at.wave * NG + at.lg) * share;         // every step < T: not the last segment
  const T* gi = static_cast<const T*>(p.gi) + at.b * p.sg_b;
  const T* dout = BACK ? static_cast<const T*>(p.dout) + at.b * p.sd_b : nullptr;
  const uint8_t* rs = RESET ? p.reset + at.b * p.sr_b : nullptr;
  const int groups = NG - 1 - at.lg;
  // uniform base: the wave's first group forwards, its last one backwards
  const int wave0 = tbeg + at.wave * NG * share;
  const int64_t t0 = BACK ? (int64_t)p.T - 1 - wave0 - (NG - 1) * (int64_t)share : wave0;
  const int64_t lane_t = (BACK ? groups : at.lg) * (int64_t)share;
  const uint32_t off_z = at.ok ? (uint32_t)((lane_t * p.sg_t + at.j) * sizeof(T)) : kOffNone;
  const uint32_t off_n = at.ok ? off_z + (uint32_t)(p.H * sizeof(T)) : kOffNone;
  const uint32_t off_d = BACK && at.ok ? (uint32_t)((lane_t * p.sd_t + at.j) * sizeof(T)) : kOffNone;
  struct Set {
    typename P::Raw z[U], x[U];
    unsigned int r[U];
  };
  auto load = [&](int i0, Set& s) __attribute__((always_inline)) {
    const int rem = share - i0;
    const int64_t t = BACK ? t0 - i0 : t0 + i0;
    load_steps<T, V, U, BACK, false>(gi + t * p.sg_t, p.sg_t, off_z, rem, s.z);
    if constexpr (BACK)
      load_steps<T, V, U, BACK, false>(dout + t * p.sd_t, p.sd_t, off_d, rem, s.x);
    else
      load_steps<T, V, U, BACK, false>(gi + t * p.sg_t, p.sg_t, off_n, rem, s.x);
    if constexpr (RESET) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int64_t step = BACK ? (int64_t)p.T - 1 - first - i0 - i : (int64_t)first + i0 + i;
        s.r[i] = i < rem ? rs[step * p.sr_t] : 0u;
      }
    }
  };
  Map m[V];
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = Map{1.0f, 0.0f};
  auto fold = [&](const Set& s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float gz[V], x[V];
      P::unpack(s.z[i], gz);
      P::unpack(s.x[i], x);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float z, n;
        gates<TANH && !BACK>(gz[v], x[v], z, n);
        Map e{z, BACK ? z * n : __builtin_fmaf(-z, n, n)};
        if (RESET && s.r[i]) e = Map{-0.0f, BACK ? 0.0f : e.b};
        m[v] = then<RESET>(m[v], e);
      }
    }
  };
  Set s0, s1;
  load(0, s0);
  for (int i0 = 0; i0 < share; i0 += 2 * U) {
    load(i0 + U, s1);
    fold(s0);
    if (i0 + U >= share) break;
    load(i0 + 2 * U, s0);
    fold(s1);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int d = 1; d < NG; d *= 2) {
      const Map o{__shfl_up(m[v].a, d * LC), __shfl_up(m[v].b, d * LC)};
      if (at.lg >= d) m[v] = then<RESET>(o, m[v]);
    }
  }
  if (at.lg == NG - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) lds[at.wave][at.lc * V + v] = m[v];
  }
  __syncthreads();
  if (at.wave == 0 && at.lg == 0 && at.ok) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      Map r = lds[0][at.lc * V + v];
#pragma unroll
      for (int w = 1; w < NW; ++w) r = then<RESET>(r, lds[w][at.lc * V + v]);
      p.agg[((int64_t)blockIdx.y * p.B + at.b) * p.H + at.j + v] = f2v{r.a, r.b};
    }
  }
}

// One step for each row of a batch of requests, whose states are rows of a cache.
struct StepParams {
  const void* gi;
  float* state;
  const int32_t* slots;
  void* out;
  int64_t sg_b, ss, so_b;
  int B, H, S;
};

template <typename T, bool TANH>
__global__ __launch_bounds__(256) void glr_step_kernel(StepParams p) {
  const int j = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
  if (j >= p.H) return;
  const int slot = p.slots ? p.slots[b] : b;
  const T* g = static_cast<const T*>(p.gi) + b * p.sg_b + j;
  T* o = static_cast<T*>(p.out) + b * p.so_b + j;
  if (slot < 0 || slot >= p.S) {
    *o = (T)(slot < 0 ? 0.0f : __builtin_nanf(""));
    return;
  }
  float z, n;
  gates<TANH>((float)g[0], (float)g[p.H], z, n);
  float* s = p.state + slot * p.ss + j;
  const float h = __builtin_fmaf(z, *s, __builtin_fmaf(-z, n, n));
  *s = h;
  *o = (T)h;
}

// ---- host ---------------------------------------------------------------------------

constexpr int kMaxSegments = 64;

// How a call is laid out. V channels a lane; `narrow`: 16 lanes of channels by 4
// step groups in 8 waves, tiles of 256 steps; otherwise 64 lanes of channels in
// one wave, tiles of 8 steps. `segments` walk the axis at once.
struct Plan {
  int v;
  bool narrow;
  int blocks, segments, seg;
};

constexpr int kNarrowTile = 4 * 8 * 8;

Plan make_plan(int64_t T, int64_t B, int64_t H, int v, bool can_narrow) {
  Plan r;
  r.v = v;
  r.narrow = can_narrow && T > 16 && B * ((H + 64 * v - 1) / (64 * v)) < 4096;
  const int lanes = r.narrow ? 16 : 64;
  r.blocks = (int)((H + lanes * v - 1) / (lanes * v));
  const int64_t groups = B * r.blocks;
  r.segments = 1;
  r.seg = (int)T;
  if (r.narrow) {
    const int64_t tiles = (T + kNarrowTile - 1) / kNarrowTile;
    int64_t want = std::min<int64_t>({(512 + groups - 1) / groups, tiles / 2, kMaxSegments});
    if (groups >= 192) want = 1;
    if (want > 1) {
      const int64_t per = (tiles + want - 1) / want;
      r.seg = (int)(per * kNarrowTile);
      r.segments = (int)((T + r.seg - 1) / r.seg);
    }
  }
  return r;
}

bool unit_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

int check_sizes(const char* who, int64_t T, int64_t B, int64_t H, int dtype, int activation) {
  if (T < 1) return set_error(GS_ERR_INVALID, "%s: seq length T must be > 0; got T=%lld", who, (long long)T);
  if (B < 1) return set_error(GS_ERR_INVALID, "%s: batch size B must be > 0; got B=%lld", who, (long long)B);
  if (H < 1) return set_error(GS_ERR_INVALID, "%s: hidden size H must be > 0; got H=%lld", who, (long long)H);
  if (T > (1ll << 30) || B > (1ll << 24) || H > (1ll << 20))
    return set_error(GS_ERR_INVALID, "%s: T/B/H out of supported range (T=%lld, B=%lld, H=%lld)", who, (long long)T,
                     (long long)B, (long long)H);
  if (dtype != GS_DTYPE_F32 && dtype != GS_DTYPE_BF16)
    return set_error(GS_ERR_INVALID, "%s: unknown dtype %d", who, dtype);
  if (activation != GS_ACT_NONE && activation != GS_ACT_TANH)
    return set_error(GS_ERR_INVALID, "%s: activation must be none or tanh; got %d", who, activation);
  return GS_OK;
}

// Rows of `n` elements at t * st + b * sb: written ones must not overlap each other.
int check_rows(const char* who, const char* name, int64_t T, int64_t B, int64_t n, int64_t st, int64_t sb, bool written) {
  if (st < 0 || sb < 0)
    return set_error(GS_ERR_INVALID, "%s: %s has a negative stride (%lld, %lld)", who, name, (long long)st,
                     (long long)sb);
  if (written && ((B > 1 && T > 1 && !(st >= sb * (B - 1) + n && sb >= n) && !(sb >= st * (T - 1) + n && st >= n)) ||
                  (B > 1 && sb < n) || (T > 1 && st < n)))
    return set_error(GS_ERR_INVALID, "%s: %s rows overlap (strides %lld, %lld)", who, name, (long long)st,
                     (long long)sb);
  return GS_OK;
}

// The largest lane offset of the narrow layout has to stay below 2^31 bytes: three
// groups of 8 steps apart, or of a share of a segment.
bool narrow_reach(int64_t st, int64_t groups_apart, int64_t H, int size) {
  return st < (int64_t(1) << 40) && (3 * groups_apart * st + 2 * H + 64) * size < (int64_t(1) << 31);
}

typedef void (*GlrFn)(GlrParams);
template <typename T, int V, bool NARROW>
struct Kernels {
  static constexpr int LC = NARROW ? 16 : 64, NW = NARROW ? 8 : 1, U = 8;
  template <bool TANH, bool RESET>
  static GlrFn pick(int what) {
    if (what == 0) return glr_fwd_kernel<T, V, LC, NW, U, TANH, RESET>;
    if (what == 1) return glr_bwd_kernel<T, V, LC, NW, U, TANH, RESET>;
    if constexpr (NARROW) {
      if (what == 2) return glr_segment_kernel<T, V, LC, NW, U, TANH, RESET, false>;
      if (what == 3) return glr_segment_kernel<T, V, LC, NW, U, false, RESET, true>;
    }
    return nullptr;
  }
  static GlrFn get(int what, bool tanh, bool reset) {
    return tanh ? (reset ? pick<true, true>(what) : pick<true, false>(what))
                : (reset ? pick<false, true>(what) : pick<false, false>(what));
  }
};

GlrFn kernel_of(int dtype, const Plan& plan, int what, bool tanh, bool reset) {
  if (dtype == GS_DTYPE_F32)
    return plan.narrow ? Kernels<float, 1, true>::get(what, tanh, reset) : Kernels<float, 1, false>::get(what, tanh, reset);
  if (plan.v == 2)
    return plan.narrow ? Kernels<__bf16, 2, true>::get(what, tanh, reset) : Kernels<__bf16, 2, false>::get(what, tanh, reset);
  return plan.narrow ? Kernels<__bf16, 1, true>::get(what, tanh, reset) : Kernels<__bf16, 1, false>::get(what, tanh, reset);
}

struct Strided {
  const void* p;
  int64_t st, sb;
};

Plan plan_of(int dtype, int64_t T, int64_t B, int64_t H, const Strided* t, int count) {
  const int size = dtype == GS_DTYPE_F32 ? 4 : 2;
  int v = dtype == GS_DTYPE_F32 || H % 2 ? 1 : 2;
  bool narrow = true;
  for (int i = 0; i < count; ++i) {
    if (v == 2 && (!unit_aligned(t[i].p, 4) || t[i].st % 2 || t[i].sb % 2)) v = 1;
    narrow = narrow && narrow_reach(t[i].st, 8, H, size);
  }
  Plan plan = make_plan(T, B, H, v, narrow);
  for (int i = 0; i < count && plan.segments > 1; ++i)
    if (!narrow_reach(t[i].st, plan.seg / 32, H, size)) {
      plan.segments = 1;
      plan.seg = (int)T;
    }
  return plan;
}

int64_t scratch_of(const Plan& plan, int64_t B, int64_t H) {
  return plan.segments > 1 ? (int64_t)(plan.segments - 1) * B * H * (int64_t)sizeof(f2v) : 0;
}

// What a call of these sizes may need, whatever its pointers and strides.
int64_t scratch_most(int64_t T, int64_t B, int64_t H) {
  return std::max(scratch_of(make_plan(T, B, H, 1, true), B, H), scratch_of(make_plan(T, B, H, 2, true), B, H));
}

int launch(const char* who, int dtype, const Plan& plan, GlrParams& p, bool back, bool tanh, void* scratch,
           int64_t scratch_bytes, hipStream_t stream) {
  const int64_t need = scratch_of(plan, p.B, p.H);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need || !unit_aligned(scratch, 256)))
    return set_error(GS_ERR_INVALID, "%s: scratch of %lld bytes, 256-byte aligned, required; got %lld at %p", who,
                     (long long)need, (long long)scratch_bytes, scratch);
  p.agg = static_cast<f2v*>(scratch);
  p.blocks = plan.blocks;
  p.seg = plan.seg;
  const int64_t groups = ((int64_t)p.B * plan.blocks + 7) / 8 * 8;
  if (groups * (plan.narrow ? 512 : 64) > UINT32_MAX)
    return set_error(GS_ERR_INVALID, "%s: too many channels (B=%d, H=%d)", who, p.B, p.H);
  const dim3 threads(plan.narrow ? 512 : 64);
  const bool reset = p.reset != nullptr;
  if (plan.segments > 1) {
    GlrFn fn = kernel_of(dtype, plan, back ? 3 : 2, tanh, reset);
    hipLaunchKernelGGL(fn, dim3((unsigned)groups, (unsigned)(plan.segments - 1)), threads, 0, stream, p);
    GS_CHECK_HIP(hipGetLastError());
  }
  GlrFn fn = kernel_of(dtype, plan, back ? 1 : 0, tanh, reset);
  hipLaunchKernelGGL(fn, dim3((unsigned)groups, (unsigned)plan.segments), threads, 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}

int check_fwd(const gs_glr_args* a, const char* who) {
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  int rc = check_sizes(who, a->T, a->B, a->H, a->dtype, a->activation);
  if (rc) return rc;
  if ((rc = check_rows(who, "gi", a->T, a->B, 2 * a->H, a->sg_t, a->sg_b, false))) return rc;
  if ((rc = check_rows(who, "out", a->T, a->B, a->H, a->so_t, a->so_b, true))) return rc;
  if (a->sh0_b < 0 || a->sr_t < 0 || a->sr_b < 0)
    return set_error(GS_ERR_INVALID, "%s: h0 or reset has a negative stride", who);
  return GS_OK;
}

int check_bwd(const gs_glr_bwd_args* a, const char* who) {
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  int rc = check_sizes(who, a->T, a->B, a->H, a->dtype, a->activation);
  if (rc) return rc;
  if ((rc = check_rows(who, "gi", a->T, a->B, 2 * a->H, a->sg_t, a->sg_b, false))) return rc;
  if ((rc = check_rows(who, "out", a->T, a->B, a->H, a->so_t, a->so_b, false))) return rc;
  if ((rc = check_rows(who, "dout", a->T, a->B, a->H, a->sd_t, a->sd_b, false))) return rc;
  if ((rc = check_rows(who, "dgi", a->T, a->B, 2 * a->H, a->sdg_t, a->sdg_b, true))) return rc;
  if (a->sh0_b < 0 || a->sr_t < 0 || a->sr_b < 0)
    return set_error(GS_ERR_INVALID, "%s: h0 or reset has a negative stride", who);
  return GS_OK;
}

Plan plan_fwd(const gs_glr_args* a) {
  const Strided t[2] = {{a->gi, a->sg_t, a->sg_b}, {a->out, a->so_t, a->so_b}};
  return plan_of(a->dtype, a->T, a->B, a->H, t, 2);
}

Plan plan_bwd(const gs_glr_bwd_args* a) {
  const Strided t[4] = {{a->gi, a->sg_t, a->sg_b}, {a->out, a->so_t, a->so_b}, {a->dout, a->sd_t, a->sd_b},
                        {a->dgi, a->sdg_t, a->sdg_b}};
  return plan_of(a->dtype, a->T, a->B, a->H, t, 4);
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int64_t gs_glr_scratch_bytes(const gs_glr_args* a) {
  clear_error();
  const int rc = check_fwd(a, "gs_glr_scratch_bytes");
  return rc ? rc : scratch_most(a->T, a->B, a->H);
}

extern "C" int gs_glr_fwd(const gs_glr_args* a, hipStream_t stream) {
  const char* who = "gs_glr_fwd";
  clear_error();
  const int rc = check_fwd(a, who);
  if (rc) return rc;
  if (!a->gi || !a->out) return set_error(GS_ERR_INVALID, "%s: gi and out must be non-NULL device pointers", who);
  GlrParams p{};
  p.gi = a->gi;
  p.h0 = a->h0;
  p.reset = a->reset;
  p.out = a->out;
  p.h_last = a->h_last;
  p.sg_t = a->sg_t;
  p.sg_b = a->sg_b;
  p.sh0_b = a->sh0_b;
  p.sr_t = a->sr_t;
  p.sr_b = a->sr_b;
  p.so_t = a->so_t;
  p.so_b = a->so_b;
  p.T = (int)a->T;
  p.B = (int)a->B;
  p.H = (int)a->H;
  return launch(who, a->dtype, plan_fwd(a), p, false, a->activation == GS_ACT_TANH, a->scratch, a->scratch_bytes, stream);
}

extern "C" int64_t gs_glr_bwd_scratch_bytes(const gs_glr_bwd_args* a) {
  clear_error();
  const int rc = check_bwd(a, "gs_glr_bwd_scratch_bytes");
  return rc ? rc : scratch_most(a->T, a->B, a->H);
}

extern "C" int gs_glr_bwd(const gs_glr_bwd_args* a, hipStream_t stream) {
  const char* who = "gs_glr_bwd";
  clear_error();
  const int rc = check_bwd(a, who);
  if (rc) return rc;
  if (!a->gi || !a->out || !a->dout || !a->dgi)
    return set_error(GS_ERR_INVALID, "%s: gi, out, dout and dgi must be non-NULL device pointers", who);
  GlrParams p{};
  p.gi = a->gi;
  p.h0 = a->h0;
  p.reset = a->reset;
  p.out = const_cast<void*>(a->out);
  p.dout = a->dout;
  p.dh_last = a->dh_last;
  p.dgi = a->dgi;
  p.dh0 = a->dh0;
  p.sg_t = a->sg_t;
  p.sg_b = a->sg_b;
  p.sh0_b = a->sh0_b;
  p.sr_t = a->sr_t;
  p.sr_b = a->sr_b;
  p.so_t = a->so_t;
  p.so_b = a->so_b;
  p.sd_t = a->sd_t;
  p.sd_b = a->sd_b;
  p.sdg_t = a->sdg_t;
  p.sdg_b = a->sdg_b;
  p.T = (int)a->T;
  p.B = (int)a->B;
  p.H = (int)a->H;
  return launch(who, a->dtype, plan_bwd(a), p, true, a->activation == GS_ACT_TANH, a->scratch, a->scratch_bytes, stream);
}

extern "C" int gs_glr_step(const gs_glr_step_args* a, hipStream_t stream) {
  const char* who = "gs_glr_step";
  clear_error();
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  const int rc = check_sizes(who, 1, a->B, a->H, a->dtype, a->activation);
  if (rc) return rc;
  if (!a->gi || !a->state || !a->out)
    return set_error(GS_ERR_INVALID, "%s: gi, state and out must be non-NULL device pointers", who);
  if (a->S < 1 || a->S > (1ll << 30) || (a->slots == nullptr && a->S < a->B))
    return set_error(GS_ERR_INVALID, "%s: a cache of S=%lld states does not hold B=%lld rows", who, (long long)a->S,
                     (long long)a->B);
  if (a->sg_b < 0 || (a->S > 1 && a->ss < a->H) || (a->B > 1 && a->so_b < a->H))
    return set_error(GS_ERR_INVALID, "%s: strides (gi %lld, state %lld, out %lld) do not describe rows of H=%lld", who,
                     (long long)a->sg_b, (long long)a->ss, (long long)a->so_b, (long long)a->H);
  if (a->B > 65535) return set_error(GS_ERR_INVALID, "%s: B=%lld exceeds 65535", who, (long long)a->B);
  StepParams p{a->gi, a->state, a->slots, a->out, a->sg_b, a->ss, a->so_b, (int)a->B, (int)a->H, (int)a->S};
  const bool tanh = a->activation == GS_ACT_TANH;
  auto fn = a->dtype == GS_DTYPE_F32 ? (tanh ? glr_step_kernel<float, true> : glr_step_kernel<float, false>)
                                     : (tanh ? glr_step_kernel<__bf16, true> : glr_step_kernel<__bf16, false>);
  hipLaunchKernelGGL(fn, dim3((unsigned)((a->H + 255) / 256), (unsigned)a->B), dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}
