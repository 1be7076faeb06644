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
// the sizes, so results are reproducible. With few channels and a long axis a workgroup
// takes one tile instead, and tiles hand their states on through memory (see chain()).
//
// Bound by memory where there are enough waves: T 256, B 64, H 2048 in bf16 takes 37 us
// forward and 77 backward, 5.4 and 5.2 TB/s where a copy reaches 5.2; T 512, B 16, H 512 in
// fp32 11 and 19 (4.5, 5.4). The chained layouts reach 3.3 to 5.6: T 4096, B 8, H 1024
// in bf16 46 and 84 us (in a training step, with its memory cold, 50 to 53 and 88), T 65536,
// B 1, H 1024 121 and 193, in fp32 172 and 287, and 5 us each before them to clear the chain's
// words. What keeps them below a copy is the start of each workgroup (its ticket, its loads
// and the wait for its carry, one after the other), which six waves a SIMD only partly hide;
// and, forwards in bf16, rows of 64 bytes a workgroup.
#include "gs_mfma.h"

namespace gs {
namespace {

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
  uint64_t* maps;      // chained layout only: see Chain
  uint32_t* states;
  uint32_t* tickets;
  uint32_t* fault;     // host-visible word, or NULL: see chain()
  int64_t sg_t, sg_b, sh0_b, sr_t, sr_b, so_t, so_b, sd_t, sd_b, sdg_t, sdg_b;
  int T, B, H;
  int blocks;          // channel blocks per batch row
  int tiles;           // chained layout: tiles of the time axis
  int polls;           // chained layout: bound of a workgroup's polls
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
// A map of many steps keeps a > 0: a product of z under the smallest float is held as that,
// so that an infinite state, which no step takes away, does not become 0 x infinity (a finite
// one moves by less than 1.5e-45 of its size). As unsigned words -0 and NaNs are above it.
__device__ __forceinline__ float span_a(float a) { return __uint_as_float(max(__float_as_uint(a), 1u)); }
template <bool RESET>
__device__ __forceinline__ Map then_span(const Map& first, const Map& second) {
  Map r = then<RESET>(first, second);
  r.a = span_a(r.a);
  return r;
}

// V elements of type T in one buffer access: an fp32, a bf16 or two of those.
template <typename T, int V>
struct Pack {
  static constexpr int kBytes = V * (int)sizeof(T);
  static_assert(kBytes == 2 || kBytes == 4, "2 or 4 bytes a lane");
  typedef unsigned int Raw;
  static __device__ __forceinline__ Raw load(const void* base, uint32_t off) {
    const auto r = bounded_rsrc(base, 0x7fffffffu);
    if constexpr (kBytes == 2)
      return (unsigned int)(unsigned short)__builtin_amdgcn_raw_buffer_load_b16(r, (int)off, 0, 0);
    else
      return __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0);
  }
  static __device__ __forceinline__ void store(void* base, uint32_t off, const float (&x)[V]) {
    const auto r = bounded_rsrc(base, 0x7fffffffu);
    if constexpr (kBytes == 2)
      __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, (__bf16)x[0]), r, (int)off, 0, 0);
    else if constexpr (V == 1)
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[0]), r, (int)off, 0, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b32(
          __builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{x[0], x[1]}), bf2v)), r, (int)off, 0, 0);
  }
  static __device__ __forceinline__ void unpack(Raw w, float (&x)[V]) {
    if constexpr (V == 2) {
      x[0] = __uint_as_float(w << 16);
      x[1] = __uint_as_float(w & 0xffff0000u);
    } else {
      x[0] = __uint_as_float(kBytes == 2 ? w << 16 : w);
    }
  }
};

template <bool TANH>
__device__ __forceinline__ void gates(float gz, float gn, float& z, float& n) {
  z = sigmoid(gz);
  n = TANH ? tanh_near(gn) : gn;
}
// (1 - z) n in one rounding. The fma makes infinity - infinity of an infinite n (there is none
// after tanh), which stays infinite, also where z has rounded to 1; a NaN in z passes.
template <bool TANH>
__device__ __forceinline__ float candidate(float z, float n) {
  const float b = __builtin_fmaf(-z, n, n);
  return !TANH && __builtin_isinf(n) ? (1.0f + z) * n : b;
}

// Where a lane is: its channels, its step group, and its wave (uniform).
template <int V, int LC, int NW>
struct Place {
  static constexpr int NG = 64 / LC;
  int b, j, lc, lg, wave;
  int tile;      // chained layout: the workgroup's tile of the time axis
  bool ok, any;  // the lane's channels exist; the workgroup's do
  __device__ __forceinline__ void at_group(const GlrParams& p, int group) {
    b = group / p.blocks;
    any = b < p.B;
    j = ((group - b * p.blocks) * LC + lc) * V;
    ok = any && j < p.H;
  }
  // CHAIN: workgroups of one XCD (workgroup mod 8) draw their places in order, all its
  // channel blocks of a tile before those of the next, so that whatever a workgroup waits
  // for belongs to one that has started before it.
  template <bool CHAIN>
  __device__ __forceinline__ void init(const GlrParams& p, int* shared) {
    const int lane = threadIdx.x & 63;
    wave = NW > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    lc = lane % LC;
    lg = lane / LC;
    tile = 0;
    // neighbours in a row, which share cache lines, on one XCD
    const int xcd = blockIdx.x & 7;
    if constexpr (CHAIN) {
      if (threadIdx.x == 0)
        *shared = (int)__hip_atomic_fetch_add(p.tickets + 32 * xcd, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      const int ticket = __builtin_amdgcn_readfirstlane(*shared + 1);  // the counters start at -1 (or past the first tile)
      const int per = gridDim.x / p.tiles >> 3;
      tile = ticket / per;
      at_group(p, xcd * per + ticket - tile * per);
      if (tile >= p.tiles) ok = any = false;  // glr_fill_kernel's second start
    } else {
      at_group(p, xcd * (int)(gridDim.x >> 3) + (int)(blockIdx.x >> 3));
    }
  }
};

// Chained layout, for few channels and a long axis: a workgroup takes one tile, and the
// state with which it starts comes from the workgroups before it in time. Each publishes
// its tile's map as soon as it has it; every kLink-th publishes the state after its tile.
// A tile's carry is then the last such state taken through the maps since, joined in order
// before the state is there, so that results do not depend on timing, and the chain of
// waits along the axis has one link in kLink tiles. Words are published with one 64-bit
// (map) or 32-bit (state) store and are all ones before that; NaNs are stored in one form,
// which is not all ones. A workgroup whose polls run out takes NaN for what is not there and says
// so in the host's fault word, so that a launch ends whatever happens and the host can tell why its
// results are NaN.
constexpr int kLink = 16;
constexpr uint32_t kNaN = 0x7fc00000u, kNone32 = 0xffffffffu;
constexpr uint64_t kNone64 = ~uint64_t(0);
constexpr int kMostPolls = 1 << 22;  // seconds

__device__ __forceinline__ uint32_t word_of(float x) { return x != x ? kNaN : __float_as_uint(x); }

// wave 0 of a workgroup: the carry of its tile, from the map `m` of the tile (every lane of
// a channel holds it). The lane groups of a channel gather a share of the maps each.
template <int V, int LC, int NW, bool RESET>
__device__ __forceinline__ void chain(const GlrParams& p, const Place<V, LC, NW>& at, const float* first, int64_t ld,
                                      const Map (&m)[V], float (&carry)[V], float (&last)[V]) {
  constexpr int NG = 64 / LC, kShare = kLink / NG;
  static_assert(NG > 1 && kShare % 4 == 0, "a lane group's share of the maps, in fours");
  const int64_t row = (int64_t)p.blocks * LC * V, plane = (int64_t)p.B * row;
  const int s = at.tile, from = s & ~(kLink - 1), count = s - from;
  const int64_t c0 = (int64_t)at.b * row + (int64_t)at.j;
  const bool link = count == kLink - 1;
  if (at.lg == 0 && !link && s + 1 < p.tiles) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      __hip_atomic_store(p.maps + s * plane + c0 + v, (uint64_t)word_of(m[v].a) | (uint64_t)word_of(m[v].b) << 32,
                         __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // the maps of this lane group, four at a time
  const uint64_t* src = p.maps + (from + kShare * at.lg) * plane + c0;
  const int mine = count - kShare * at.lg;
  Map f[V];
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = Map{1.0f, 0.0f};
  int polls = 0;
  for (int k0 = 0; k0 < kShare && k0 < count; k0 += 4) {
    uint64_t w[4][V];
    for (;; ++polls) {
      bool ready = true;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          w[k][v] = 0u;
          if (k0 + k < mine)
            w[k][v] = __hip_atomic_load(src + (k0 + k) * plane + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          ready = ready && w[k][v] != kNone64;
        }
      if (__builtin_amdgcn_ballot_w64(!ready) == 0 || polls >= p.polls) break;
      __builtin_amdgcn_s_sleep(1);
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (w[k][v] == kNone64) w[k][v] = (uint64_t)kNaN << 32 | kNaN;
        const Map x{__uint_as_float((uint32_t)w[k][v]), __uint_as_float((uint32_t)(w[k][v] >> 32))};
        if (k0 + k < mine) f[v] = then_span<RESET>(f[v], x);
      }
  }
  // all of them in order, and this tile's: what is left once the state is there is one step
  Map all[V], past[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    all[v] = Map{__shfl(f[v].a, at.lc), __shfl(f[v].b, at.lc)};
#pragma unroll
    for (int g = 1; g < NG; ++g) all[v] = then_span<RESET>(all[v], Map{__shfl(f[v].a, g * LC + at.lc), __shfl(f[v].b, g * LC + at.lc)});
    past[v] = then_span<RESET>(all[v], m[v]);
  }
  uint32_t h[V];
  if (from) {
    const uint32_t* state = p.states + (s / kLink) * plane + c0;
    for (;; ++polls) {
      bool ready = true;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        h[v] = __hip_atomic_load(state + v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        ready = ready && h[v] != kNone32;
      }
      if (__builtin_amdgcn_ballot_w64(!ready) == 0 || polls >= p.polls) break;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float c = first != nullptr && at.ok ? first[(int64_t)at.b * ld + at.j + v] : 0.0f;
      h[v] = word_of(c);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float c = __uint_as_float(h[v] == kNone32 ? kNaN : h[v]);
    last[v] = apply<RESET>(past[v], c);
    if (link && s + 1 < p.tiles && at.lg == 0)
      __hip_atomic_store(p.states + (s / kLink + 1) * plane + c0 + v, word_of(last[v]), __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    carry[v] = apply<RESET>(all[v], c);
  }
  if (polls >= p.polls && p.fault != nullptr && (threadIdx.x & 63) == 0)
    __hip_atomic_store(p.fault, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

// The maps before a lane's own steps: given each lane's map of its U steps,
// returns the state at the lane's first step and advances `carry` past the tile.
// `lds` is one of two buffers used in turn: a wave writes a buffer again only
// after a barrier that every wave reaches when it has read it.
// CHAIN: the carry comes from the workgroups of the tiles before (`first`, rows of ld: the
// state with which the axis starts); `carry` is left as the state after the tile in wave 0.
template <int V, int LC, int NW, bool RESET, bool CHAIN>
__device__ __forceinline__ void enter(const GlrParams& p, const Place<V, LC, NW>& at, Map (&m)[V], float (&carry)[V],
                                      float (&h)[V], Map (*lds)[LC * V], const float* first, int64_t ld) {
  constexpr int NG = 64 / LC;
  Map before[V];
#pragma unroll
  for (int v = 0; v < V; ++v) m[v].a = span_a(m[v].a);
  if constexpr (NG > 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int d = 1; d < NG; d *= 2) {
        const Map o{__shfl_up(m[v].a, d * LC), __shfl_up(m[v].b, d * LC)};
        if (at.lg >= d) m[v] = then_span<RESET>(o, m[v]);
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
    float start[V];
    if constexpr (CHAIN) {
      if (at.wave == 0) {
        Map whole[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          whole[v] = lds[0][at.lc * V + v];
#pragma unroll
          for (int w = 1; w < NW; ++w) whole[v] = then_span<RESET>(whole[v], lds[w][at.lc * V + v]);
        }
        chain<V, LC, NW, RESET>(p, at, first, ld, whole, start, carry);
        if (at.lg == 0) {
#pragma unroll
          for (int v = 0; v < V; ++v) lds[NW][at.lc * V + v].b = start[v];
        }
      }
      lds_barrier();
#pragma unroll
      for (int v = 0; v < V; ++v) start[v] = lds[NW][at.lc * V + v].b;
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) start[v] = carry[v];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float c = start[v], mine = c;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        if (w == at.wave) mine = c;
        c = apply<RESET>(lds[w][at.lc * V + v], c);
      }
      if constexpr (!CHAIN) carry[v] = c;
      h[v] = NG > 1 ? apply<RESET>(before[v], mine) : mine;
    }
  }
}

template <int V>
__device__ __forceinline__ void first_carry(const float* first, int64_t ld, int b, int j, bool ok, float (&carry)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) carry[v] = first != nullptr && ok ? first[(int64_t)b * ld + j + v] : 0.0f;
}

// Loads of U steps. Step i of a lane is t0 + lg U + i forwards, and t0 - lg U - i
// backwards (BACK); rem is how many of its steps exist. Offsets are the lane's
// part only (its channel and its group's distance from the wave's base); the
// base moves with i and the wave, in scalar registers.
template <typename T, int V, int U, bool BACK>
__device__ __forceinline__ void load_steps(const void* base, int64_t st, uint32_t off, int rem,
                                           typename Pack<T, V>::Raw (&x)[U]) {
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const T* q = static_cast<const T*>(base) + (BACK ? -i : i) * st;
    x[i] = Pack<T, V>::load(q, i < rem ? off : kOffNone);
  }
}

__device__ __forceinline__ unsigned int load_flag(const uint8_t* base, uint32_t off) {
  return (unsigned char)__builtin_amdgcn_raw_buffer_load_b8(bounded_rsrc(base, 0x7fffffffu), (int)off, 0, 0);
}

template <typename T, int V, int LC, int NW, int U, bool TANH, bool RESET, bool CHAIN>
__global__ __launch_bounds__(64 * NW, CHAIN ? 6 : 1) void glr_fwd_kernel(GlrParams p) {
  typedef Pack<T, V> P;
  constexpr int NG = 64 / LC, kTile = NG * NW * U;
  __shared__ Map lds[CHAIN ? 1 : 2][NW > 1 ? NW + CHAIN : 1][LC * V];
  __shared__ int ticket;
  Place<V, LC, NW> at;
  at.template init<CHAIN>(p, &ticket);
  if (!at.any) return;  // uniform
  float carry[V];
  if constexpr (!CHAIN) first_carry<V>(p.h0, p.sh0_b, at.b, at.j, at.ok, carry);

  const T* gi = static_cast<const T*>(p.gi) + at.b * p.sg_b;
  T* out = static_cast<T*>(p.out) + at.b * p.so_b;
  const uint8_t* rs = RESET ? p.reset + at.b * p.sr_b : nullptr;
  const uint32_t lane_g = (uint32_t)((at.lg * U * p.sg_t + at.j) * sizeof(T));
  const uint32_t off_z = at.ok ? lane_g : kOffNone;
  const uint32_t off_n = at.ok ? lane_g + (uint32_t)(p.H * sizeof(T)) : kOffNone;
  const uint32_t off_o = at.ok ? (uint32_t)((at.lg * U * p.so_t + at.j) * sizeof(T)) : kOffNone;
  const uint32_t off_r = (uint32_t)(at.lg * U * p.sr_t);
  struct Set {
    typename P::Raw z[U], n[U];
    unsigned int r[U];
  };
  auto load = [&](int t0, Set& s) __attribute__((always_inline)) {
    const int tw = t0 + at.wave * NG * U;  // the wave's first step
    const T* g = gi + tw * p.sg_t;
    const int rem = p.T - tw - at.lg * U;
    load_steps<T, V, U, false>(g, p.sg_t, off_z, rem, s.z);
    load_steps<T, V, U, false>(g, p.sg_t, off_n, rem, s.n);
    if constexpr (RESET) {
#pragma unroll
      for (int i = 0; i < U; ++i) s.r[i] = load_flag(rs + (tw + i) * p.sr_t, i < rem ? off_r : kOffNone);
    }
  };
  auto tile = [&](int t0, const Set& s, Map (*buf)[LC * V]) __attribute__((always_inline)) {
    const int tw = t0 + at.wave * NG * U;
    const int rem = p.T - tw - at.lg * U;
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
        e[i][v] = Map{z, candidate<TANH>(z, n)};
        if (RESET && s.r[i]) e[i][v].a = -0.0f;
        if (i >= rem) e[i][v] = Map{1.0f, 0.0f};
        m[v] = then<RESET>(m[v], e[i][v]);
      }
    }
    float h[V];
    enter<V, LC, NW, RESET, CHAIN>(p, at, m, carry, h, buf, p.h0, p.sh0_b);
    T* o = out + tw * p.so_t;
#pragma unroll
    for (int i = 0; i < U; ++i) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = apply<RESET>(e[i][v], h[v]);
      P::store(o + i * p.so_t, i < rem ? off_o : kOffNone, h);
    }
  };
  Set s0;
  if constexpr (CHAIN) {
    load(at.tile * kTile, s0);
    tile(at.tile * kTile, s0, lds[0]);
  } else {
    Set s1;
    load(0, s0);
    for (int t0 = 0; t0 < p.T; t0 += 2 * kTile) {
      load(t0 + kTile, s1);
      tile(t0, s0, lds[0]);
      if (t0 + kTile >= p.T) break;
      load(t0 + 2 * kTile, s0);
      tile(t0 + kTile, s1, lds[1]);
    }
  }
  if (p.h_last != nullptr && (!CHAIN || at.tile == p.tiles - 1) && at.ok && at.lg == 0 && at.wave == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) p.h_last[(int64_t)at.b * p.H + at.j + v] = carry[v];
  }
}

// The same walk from the last step to the first: tau = T - 1 - t counts up.
template <typename T, int V, int LC, int NW, int U, bool TANH, bool RESET, bool CHAIN>
__global__ __launch_bounds__(64 * NW) void glr_bwd_kernel(GlrParams p) {
  typedef Pack<T, V> P;
  constexpr int NG = 64 / LC, kTile = NG * NW * U;
  __shared__ Map lds[CHAIN ? 1 : 2][NW > 1 ? NW + CHAIN : 1][LC * V];
  __shared__ int ticket;
  Place<V, LC, NW> at;
  at.template init<CHAIN>(p, &ticket);
  if (!at.any) return;  // uniform
  float carry[V];
  if constexpr (!CHAIN) first_carry<V>(p.dh_last, p.H, at.b, at.j, at.ok, carry);

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
  const uint32_t off_r = (uint32_t)(back * p.sr_t);
  const uint32_t off_dz = at.ok ? lane_off(p.sdg_t) : kOffNone, off_dn = at.ok ? off_dz + off_h : kOffNone;
  struct Set {
    typename P::Raw z[U], n[U], h[U], d[U];
    unsigned int r[U];
  };
  auto load = [&](int t0, Set& s) __attribute__((always_inline)) {
    const int tw = t0 + at.wave * NG * U;  // the wave's first tau
    const int64_t t = p.T - 1 - tw - (NG - 1) * U;
    const int rem = p.T - tw - at.lg * U;
    const int before = p.T - 1 - tw - at.lg * U;  // steps before the lane's first: step i has h_{t-1} in `out` if i < before
    load_steps<T, V, U, true>(gi + t * p.sg_t, p.sg_t, off_z, rem, s.z);
    load_steps<T, V, U, true>(gi + t * p.sg_t, p.sg_t, off_n, rem, s.n);
    load_steps<T, V, U, true>(dout + t * p.sd_t, p.sd_t, off_d, rem, s.d);
    load_steps<T, V, U, true>(out + (t - 1) * p.so_t, p.so_t, off_o, min(rem, before), s.h);
    if constexpr (RESET) {
#pragma unroll
      for (int i = 0; i < U; ++i) s.r[i] = load_flag(rs + (t - i) * p.sr_t, i < rem ? off_r : kOffNone);
    }
  };
  auto tile = [&](int t0, const Set& s, Map (*buf)[LC * V]) __attribute__((always_inline)) {
    const int tw = t0 + at.wave * NG * U;
    const int rem = p.T - tw - at.lg * U;
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
    enter<V, LC, NW, RESET, CHAIN>(p, at, m, carry, E, buf, p.dh_last, p.H);
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
  Set s0;
  if constexpr (CHAIN) {
    load(at.tile * kTile, s0);
    tile(at.tile * kTile, s0, lds[0]);
  } else {
    Set s1;
    load(0, s0);
    for (int t0 = 0; t0 < p.T; t0 += 2 * kTile) {
      load(t0 + kTile, s1);
      tile(t0, s0, lds[0]);
      if (t0 + kTile >= p.T) break;
      load(t0 + 2 * kTile, s0);
      tile(t0 + kTile, s1, lds[1]);
    }
  }
  if (p.dh0 != nullptr && (!CHAIN || at.tile == p.tiles - 1) && at.ok && at.lg == 0 && at.wave == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) p.dh0[(int64_t)at.b * p.H + at.j + v] = carry[v];
  }
}

// All ones over the chain's words and counters. `start`: the counters'
// first value, before the first tile (-1) or the second, which then waits in vain.
__global__ __launch_bounds__(256) void glr_fill_kernel(u4v* p, int64_t n, uint32_t start) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  u4v w{kNone32, kNone32, kNone32, kNone32};
  if (e < 8 * 8 && e % 8 == 0) w[0] = start;  // the counters' lines
  p[e] = w;
}

// One step for each row of a batch of requests, whose states are rows of a cache: one lane a
// channel, one launch. B 8, H 1024 in bf16 takes 2.3 us on the GPU, what an empty launch takes.
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
  const float h = __builtin_fmaf(z, *s, candidate<TANH>(z, n));
  *s = h;
  *o = (T)h;
}

// ---- host ---------------------------------------------------------------------------

// The layouts: lanes of channels, waves, and whether tiles are chained. A lane holds
// kSteps steps of v channels, so a tile is kSteps x 64 / lanes x waves steps.
constexpr int kSteps = 8;
struct LayoutOf {
  int lanes, waves;
  bool chain;
};
constexpr LayoutOf kLayouts[] = {{64, 1, false}, {64, 4, false}, {32, 8, false}, {16, 8, false}, {16, 8, true}, {32, 8, true}};
constexpr int kChain = 4, kWideChain = 5;
constexpr int tile_of(int layout) { return kSteps * (64 / kLayouts[layout].lanes) * kLayouts[layout].waves; }

struct Plan {
  int v, layout, blocks, tiles;
};

int64_t groups_of(const Plan& p, int64_t B) {
  return (B * p.blocks + 7) / 8 * 8 * (kLayouts[p.layout].chain ? p.tiles : 1);
}
// A launch counts its threads in 32 bits.
bool fits_launch(const Plan& p, int64_t B) { return groups_of(p, B) * 64 * kLayouts[p.layout].waves <= UINT32_MAX; }

// Few channels leave the CUs with few waves, and a row's steps then go to more of them at
// once; many channels have their waves without that, and each layer of it (LDS, barriers,
// runs of 16 lanes in memory) costs. Measured in us, forward / backward, tanh, one layout
// after the other on the same tensors:
//   T, B, H            64 x 1       64 x 4       32 x 8       16 x 8       16 x 8 chained
//   512, 128, 1024 f32 163 / 329    166 / 338    193 / 368    238 / 503
//   256, 64, 2048 bf16 53 / 82      37 / 86      44 / 119     45 / 167
//   8192, 32, 512 f32  687 / 1345   287 / 629    359 / 756    461 / 861    320 / 672
//   512, 16, 512 f32   45 / 79      17 / 27      11 / 20      12 / 21
//   1500, 11, 512 f32  125 / 226    42 / 69      21 / 37      25 / 46      23 / 37
//   4096, 16, 512 f32  340 / 644    114 / 249    93 / 180     107 / 218    82 / 163
//   4096, 4, 512 f32   335 / 607    109 / 181    46 / 75      30 / 51      22 / 37
//   640, 8, 512 f32    54 / 98      20 / 32      11 / 17      8.3 / 16     11 / 16
//   640, 4, 512 f32    55 / 98      20 / 31      9.8 / 15     7.2 / 11     9.3 / 10
//   65536, 1, 1024 b.  11600/17400  3290 / 4960  1320 / 2080  781 / 1340   119 / 209
//   8, 1024, 1024 bf16 12 / 21      29 / 54      115 / 298    232 / 611
// The last row is the loop below: no layout whose tile is four times the row and more.
// Chained tiles of 32 lanes have whole cache lines of a step but half as many steps; they
// pay where the lines are many (backwards, and in fp32) and so are the channels:
//   T, B, H                 16 x 8 chained   32 x 8 chained
//   65536, 1, 1024 bf16     113 / 204        119 / 191
//   4096, 8, 1024 bf16      44 / 93          48 / 86
//   65536, 1, 1024 f32      178 / 357        171 / 303
//   4096, 16, 512 f32       83 / 166         79 / 149
//   40000, 1, 333 f32       49 / 106         54 / 108
Plan make_plan(int64_t T, int64_t B, int64_t H, int v, bool near, bool lines) {
  // step groups side by side that give each CU eight waves
  const double want = 131072.0 / (double)(B * ((H + v - 1) / v));
  int l = want <= 1.5 ? 0 : want <= 10 ? 1 : want <= 28 ? 2 : 3;
  while (l > 0 && tile_of(l) >= 4 * T) --l;
  auto plan = [&](int layout) {
    Plan r{v, layout, 0, 0};
    const int lanes = kLayouts[layout].lanes;
    r.blocks = (int)((H + lanes * v - 1) / (lanes * v));
    r.tiles = (int)((T + tile_of(layout) - 1) / tile_of(layout));
    return r;
  };
  if (near && want > 12 && T > (want > 48 ? 2 : 4) * tile_of(kChain)) {
    const Plan r = plan(lines && want <= 256 ? kWideChain : kChain);
    if (fits_launch(r, B)) return r;  // from T = 2^28 on, tiles make more workgroups than a launch holds
  }
  return plan(near || l < 1 ? l : 1);
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

// Where a wave's lanes hold several step groups, a lane's offset from the wave's base has
// to stay below 2^31 bytes.
bool lanes_reach(int64_t st, int64_t H, int size) {
  return st < (int64_t(1) << 40) && (3 * kSteps * st + 2 * H + 64) * size < (int64_t(1) << 31);
}

// Which scans the wide chain is for (make_plan's `lines`).
template <typename T>
constexpr bool many_lines(bool back) {
  return back || sizeof(T) == 4;
}

typedef void (*GlrFn)(GlrParams);
template <typename T, int V, int L, bool BACK, bool TANH>
GlrFn kernel_at(bool reset) {
  constexpr int LC = kLayouts[L].lanes, NW = kLayouts[L].waves;
  constexpr bool CHAIN = kLayouts[L].chain;
  if constexpr (BACK)
    return reset ? glr_bwd_kernel<T, V, LC, NW, kSteps, TANH, true, CHAIN> : glr_bwd_kernel<T, V, LC, NW, kSteps, TANH, false, CHAIN>;
  else
    return reset ? glr_fwd_kernel<T, V, LC, NW, kSteps, TANH, true, CHAIN> : glr_fwd_kernel<T, V, LC, NW, kSteps, TANH, false, CHAIN>;
}
template <typename T, int V, bool BACK, bool TANH>
GlrFn kernel_in(int layout, bool reset) {
  if constexpr (many_lines<T>(BACK))
    if (layout == kWideChain) return kernel_at<T, V, kWideChain, BACK, TANH>(reset);
  switch (layout) {
    case 0: return kernel_at<T, V, 0, BACK, TANH>(reset);
    case 1: return kernel_at<T, V, 1, BACK, TANH>(reset);
    case 2: return kernel_at<T, V, 2, BACK, TANH>(reset);
    case 3: return kernel_at<T, V, 3, BACK, TANH>(reset);
    default: return kernel_at<T, V, kChain, BACK, TANH>(reset);
  }
}
template <typename T, int V>
GlrFn kernel_for(const Plan& plan, bool back, bool tanh, bool reset) {
  return back ? (tanh ? kernel_in<T, V, true, true>(plan.layout, reset) : kernel_in<T, V, true, false>(plan.layout, reset))
              : (tanh ? kernel_in<T, V, false, true>(plan.layout, reset) : kernel_in<T, V, false, false>(plan.layout, reset));
}
GlrFn kernel_of(int dtype, const Plan& plan, bool back, bool tanh, bool reset) {
  if (dtype == GS_DTYPE_F32) return kernel_for<float, 1>(plan, back, tanh, reset);
  return plan.v == 2 ? kernel_for<__bf16, 2>(plan, back, tanh, reset) : kernel_for<__bf16, 1>(plan, back, tanh, reset);
}

struct Strided {
  const void* p;
  int64_t st, sb;
};

bool lines_of(int dtype, bool back) { return dtype == GS_DTYPE_F32 ? many_lines<float>(back) : many_lines<__bf16>(back); }

Plan plan_of(int dtype, bool back, int64_t T, int64_t B, int64_t H, const Strided* t, int count, int64_t sr_t) {
  const int size = dtype == GS_DTYPE_F32 ? 4 : 2;
  int v = dtype == GS_DTYPE_F32 || H % 2 ? 1 : 2;
  bool near = true;
  for (int i = 0; i < count; ++i) {
    if (v == 2 && (!unit_aligned(t[i].p, 4) || t[i].st % 2 || t[i].sb % 2)) v = 1;
    near = near && lanes_reach(t[i].st, H, size);
  }
  return make_plan(T, B, H, v, near && lanes_reach(sr_t, 0, 1), lines_of(dtype, back));
}

// The chain's scratch: eight counters on lines of their own, the maps, the states.
constexpr int64_t kTicketBytes = 8 * 32 * 4;
struct ChainBytes {
  int64_t maps = 0, states = 0, total = 0;  // offsets
};
ChainBytes chain_bytes(const Plan& plan, int64_t B) {
  ChainBytes c;
  if (!kLayouts[plan.layout].chain) return c;
  const int64_t plane = B * plan.blocks * kLayouts[plan.layout].lanes * plan.v;
  c.maps = kTicketBytes;
  c.states = c.maps + align256(plan.tiles * plane * 8);
  c.total = c.states + align256((plan.tiles / kLink + 1) * plane * 4);
  return c;
}

// What a call of these sizes may need, whatever its pointers and strides.
int64_t scratch_most(int dtype, bool back, int64_t T, int64_t B, int64_t H) {
  const bool lines = lines_of(dtype, back);
  const int64_t one = chain_bytes(make_plan(T, B, H, 1, true, lines), B).total;
  return dtype == GS_DTYPE_F32 ? one : std::max(one, chain_bytes(make_plan(T, B, H, 2, true, lines), B).total);
}

int launch(const char* who, int dtype, const Plan& plan, GlrParams& p, bool back, bool tanh, void* scratch,
           int64_t scratch_bytes, uint32_t* fault_mirror, int32_t poll_limit, hipStream_t stream) {
  if (!fits_launch(plan, p.B))
    return set_error(GS_ERR_INVALID, "%s: more workgroups than a launch holds (T=%d, B=%d, H=%d)", who, p.T, p.B, p.H);
  const ChainBytes c = chain_bytes(plan, p.B);
  if (c.total > 0 && (scratch == nullptr || scratch_bytes < c.total || !unit_aligned(scratch, 256)))
    return set_error(GS_ERR_INVALID, "%s: scratch of %lld bytes, 256-byte aligned, required; got %lld at %p", who,
                     (long long)c.total, (long long)scratch_bytes, scratch);
  p.blocks = plan.blocks;
  p.tiles = plan.tiles;
  p.fault = fault_mirror;
  p.polls = poll_limit ? (int)std::min<int64_t>(std::abs((int64_t)poll_limit), INT32_MAX) : kMostPolls;
  const int threads = 64 * kLayouts[plan.layout].waves;
  const int64_t groups = groups_of(plan, p.B);
  if (c.total > 0) {
    p.tickets = static_cast<uint32_t*>(scratch);
    p.maps = reinterpret_cast<uint64_t*>(static_cast<char*>(scratch) + c.maps);
    p.states = reinterpret_cast<uint32_t*>(static_cast<char*>(scratch) + c.states);
    const int64_t n = c.total / 16;
    const uint32_t start = kNone32 + (poll_limit < 0 ? (uint32_t)(groups / plan.tiles / 8) : 0u);
    hipLaunchKernelGGL(glr_fill_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream,
                       static_cast<u4v*>(scratch), n, start);
    GS_CHECK_HIP(hipGetLastError());
  }
  hipLaunchKernelGGL(kernel_of(dtype, plan, back, tanh, p.reset != nullptr), dim3((unsigned)groups), dim3(threads), 0,
                     stream, p);
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
  return plan_of(a->dtype, false, a->T, a->B, a->H, t, 2, a->sr_t);
}

Plan plan_bwd(const gs_glr_bwd_args* a) {
  const Strided t[4] = {{a->gi, a->sg_t, a->sg_b}, {a->out, a->so_t, a->so_b}, {a->dout, a->sd_t, a->sd_b},
                        {a->dgi, a->sdg_t, a->sdg_b}};
  return plan_of(a->dtype, true, a->T, a->B, a->H, t, 4, a->sr_t);
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int64_t gs_glr_scratch_bytes(const gs_glr_args* a) {
  clear_error();
  const int rc = check_fwd(a, "gs_glr_scratch_bytes");
  return rc ? rc : scratch_most(a->dtype, false, a->T, a->B, a->H);
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
  return launch(who, a->dtype, plan_fwd(a), p, false, a->activation == GS_ACT_TANH, a->scratch, a->scratch_bytes,
                a->fault_mirror, a->poll_limit, stream);
}

extern "C" int64_t gs_glr_bwd_scratch_bytes(const gs_glr_bwd_args* a) {
  clear_error();
  const int rc = check_bwd(a, "gs_glr_bwd_scratch_bytes");
  return rc ? rc : scratch_most(a->dtype, true, a->T, a->B, a->H);
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
  return launch(who, a->dtype, plan_bwd(a), p, true, a->activation == GS_ACT_TANH, a->scratch, a->scratch_bytes,
                a->fault_mirror, a->poll_limit, stream);
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
