// Selective state space scan (gfx950): a recurrence whose decay depends on its input,
//   dt = softplus(delta + delta_bias),  a[n] = exp(dt A[c][n]),
//   h_t[n] = a[n] h_{t-1}[n] + dt u B_t[n],  y = sum_n C_t[n] h_t[n] + D u,  out = y silu(z),
// for every channel c of a batch row with N states each; B and C are shared by the channels.
// reset[t][b] != 0 starts a new sequence at step t: h_{t-1} is taken as 0, whatever it holds.
//
// Backward, with G_t[n] the gradient of h_t[n] and dy that of y:
//   G_t = C_t dy + a_{t+1} G_{t+1},  dC_t[n] = sum_c h_t[n] dy,  dB_t[n] = sum_c G_t[n] dt u,
//   S = sum_n G_t[n] B_t[n],  q[n] = G_t[n] a_t[n] h_{t-1}[n],
//   du = dt S + D dy,  ddt = u S + sum_n q[n] A[n],  dA[n] = sum_t q[n] dt,  dD = sum_t u dy.
//
// Layout: a lane is a channel, 64 channels of one batch row a wave, and steps come in tiles of 16. Two forms of
// the forward and of the launch that finds ends (make_plan says when each):
//   * States over the waves of a workgroup, two each (four of 32): a wave loads the rows of its steps of a
//     tile, computes what the states share (softplus, the gate) and leaves it in LDS; every wave runs its states
//     over the tile, one exponential a state and step, and leaves its part of y; each sums its steps' parts.
//   * Waves that share nothing: one has all states of its channels, and reads B and C from LDS.
// With few channels the time axis is cut into chunks. The first launch scans the first chunk and finds what each
// one between it and the last makes of a zero state; the second joins those along the axis; the
// third scans the others from their states. A training forward keeps the state before every tile, and the outputs
// before their gate, which the backward would need sums over the states (and waits) for. The backward
// finds what chunks send back, joins that, and runs each tile's steps again, forwards and then back.
// Sums over channels (dB, dC) are those of the workgroup's 64 in registers, then of the workgroups in order
// through memory: results are reproducible.
//
// Bound by the vector ALU and its exponentials: forwards 16 states at a step take some 6 instructions and an exponential each,
// every step a softplus. Measured, T 4096, B 8, H 1024, N 16 bf16: forward 139 us for the first
// launch and 174 with what is kept, ends 116, backward 540 (its VALU busy for 77 % by its counters, LDS for 43; 747 MB take
// 145 at a copy's rate); T 65536, B 1, H 1024 forward 277 + 30 + 324 (540 MB: 105), the VALU busy for 90 and 87 %;
// T 512, B 16, H 512 fp32 training 24 + 27 forward, 23 + 69 backward and 14 of joins and sums.
#include "gs_seq.h"

namespace gs {
namespace {

constexpr int kTile = 16;  // steps of a tile, and between kept states
constexpr float kLn2 = 0.6931471805599453f;

struct SsmParams {
  const void *u, *delta, *z, *bm, *cm;
  const float *A, *D, *bias, *h0;
  const uint8_t* reset;
  void* y;             // forward
  float* h_last;
  float* saved;        // [ceil(T / kTile)][B][N][H]: forward written (or NULL), backward read
  float* ungated;      // [T][B][H]: y before its gate, kept with them where there is one, else NULL
  float* ends;         // [chunks][B][N][H]: see ssm_join_kernel
  float* span;         // [2][chunks][B][H]: sum of dt over a chunk, -1 where it holds a reset; the largest dt
  const void* dy;      // backward only from here
  const float* dh_last;
  void *du, *ddelta, *dz;
  float* dh0;
  float* part_bc;      // [blocks][T][B][2N]
  float* part_a;       // [chunks][B][N + 2][H]
  int64_t su_t, su_b, sdl_t, sdl_b, sz_t, sz_b, sb_t, sb_b, sc_t, sc_b, sr_t, sr_b, sy_t, sy_b, sdy_t, sdy_b;
  int64_t sdu_t, sdu_b, sdd_t, sdd_b, sdz_t, sdz_b;
  int T, B, H, N;
  int blocks;          // channel blocks of 64
  int chunks, length;  // of the time axis, in steps
  int each;            // backward: parts of a chunk whose ends are found one by one
};

// The kernel's arguments, read anew from memory wherever this is called: kept in scalar
// registers throughout, forty strides and pointers would be spilled to lanes of vector ones.
typedef const __attribute__((address_space(4))) SsmParams* Args;
__device__ __forceinline__ Args args() {
  Args p = (Args)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// Where a workgroup is.
struct At {
  int block, b, chunk, lane, wave, ch, t0, t1;
  bool ok;  // the lane's channel exists
  // `first`: the chunk of the launch's first workgroups; `length`: of a chunk
  __device__ __forceinline__ At(const SsmParams& p, int first, int length) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int g = blockIdx.x;
    block = g % p.blocks;
    g /= p.blocks;
    b = g % p.B;
    chunk = first + g / p.B;
    ch = block * 64 + lane;
    ok = ch < p.H;
    t0 = chunk * length;
    t1 = min(p.T, t0 + length);
  }
};

template <typename T>
__device__ __forceinline__ uint32_t lane_off(const At& at) {
  return at.ok ? (uint32_t)(at.ch * (int)sizeof(T)) : kOffNone;
}
// Row t of batch row b. One past the axis is only named, with an offset that reads and writes nothing.
template <typename T>
__device__ __forceinline__ T* row_of(const void* base, int64_t st, int64_t sb, int t, int b) {
  return const_cast<T*>(static_cast<const T*>(base)) + t * st + b * sb;
}

// The flags of kTile steps from t0 on, a lane each, and as a bit mask.
__device__ __forceinline__ bool load_flag(Args p, const At& at, int t0) {
  if (p->reset == nullptr) return false;
  return at.lane < kTile && t0 + at.lane < at.t1 && p->reset[(t0 + at.lane) * p->sr_t + at.b * p->sr_b] != 0;
}
__device__ __forceinline__ uint32_t mask_of(bool flag) { return (uint32_t)__builtin_amdgcn_ballot_w64(flag); }

// B and C of a tile as floats, a wave's P states side by side; zero where there is no step or state.
typedef float f4v __attribute__((ext_vector_type(4)));
// B, then C of a wave's P states. Read in accesses of 16 bytes, whose offsets are part of the
// instruction: shorter ones in pairs need a register for the address of every fourth step.
template <int P>
struct alignas(16) Pair {
  float x[2 * P];
  __device__ __forceinline__ void read(float (&b)[P], float (&c)[P]) const {
    float v[2 * P];
#pragma unroll
    for (int i = 0; i < 2 * P; i += 4) {
      const f4v q = *reinterpret_cast<const f4v*>(x + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[i + k] = q[k];
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
      b[i] = v[i];
      c[i] = v[P + i];
    }
  }
};
template <typename T, int P, int NW>
struct Tile {
  static constexpr int NP = NW * P, kEach = kTile * NP, kPer = 2 * kEach / (64 * NW);
  static_assert(kEach % 64 == 0, "a wave's elements are all of B or all of C");
  unsigned int x[kPer];  // on their way
  __device__ __forceinline__ void load(Args p, const At& at, int t0) {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int first = (k * NW + at.wave) * 64;  // uniform
      const bool c = first >= kEach;
      const int e = (c ? first - kEach : first) + at.lane, s = e / NP, n = e % NP;
      const T* row = c ? row_of<T>(p->cm, p->sc_t, p->sc_b, t0, at.b) : row_of<T>(p->bm, p->sb_t, p->sb_b, t0, at.b);
      const int64_t st = c ? p->sc_t : p->sb_t;
      x[k] = 0;
      if (n < p->N && t0 + s < at.t1) x[k] = sizeof(T) == 2 ? *reinterpret_cast<const unsigned short*>(row + s * st + n)
                                                            : *reinterpret_cast<const unsigned int*>(row + s * st + n);
    }
  }
  __device__ __forceinline__ void put(const At& at, Pair<P> (*bc)[NW]) const {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int first = (k * NW + at.wave) * 64;
      const bool c = first >= kEach;
      const int e = (c ? first - kEach : first) + at.lane, s = e / NP, n = e % NP;
      bc[s][n / P].x[(c ? P : 0) + n % P] = Elem<T>::value(x[k]);
    }
  }
};

// Backward: parts of the axis whose ends are found one by one; p.each of them make a chunk.
__device__ __forceinline__ int parts_of(const SsmParams& p) {
  const int length = p.length / p.each;
  return (p.T + length - 1) / length;
}

// What steps whose sizes are `sum` together (-1: with a reset) and `most` at the largest are to the join.
__device__ __forceinline__ void put_span(Args p, int64_t at, float sum, float most) {
  p->span[at] = sum;
  p->span[at + (int64_t)p->chunks * p->each * p->B * p->H] = most;
}

// A as the exponent of 2, held finite: A of -infinity (a state that lasts a step), or a product past float32's
// range (the lowest float as a stand-in for it), would make a NaN with a step size of 0, which the steps behind
// the axis' end have. A NaN passes.
__device__ __forceinline__ float rate(float A) {
  const float r = A * kLog2e;
  return r < -3.0e38f ? -3.0e38f : r > 3.0e38f ? 3.0e38f : r;
}

// f(std::true_type) where a tile holds a reset, else f(std::false_type): uniform.
template <typename F>
__device__ __forceinline__ void with_flags(uint32_t flags, F&& f) {
  if (flags) f(std::true_type{});
  else f(std::false_type{});
}

// ---- forward ------------------------------------------------------------------------
//
// Of a cut axis the first of two launches (FIRST) scans the first chunk and finds the ends of those between
// it and the last; the second one, or the only one, scans the others.

template <int P, int NW>
struct FwdShared {
  float2 xs[kTile][64];  // dt, dt u
  Pair<P> bc[kTile][NW];
  float part[NW][kTile][64];
};

// OUT: the scan itself. Otherwise what a chunk makes of a zero state, and its sum of dt.
// PAD: N is not P NW; states that do not exist are left out.
template <typename T, int P, int NW, bool PAD, bool OUT>
__device__ __forceinline__ void fwd_chunk(const At& at, FwdShared<P, NW>& lds) {
  typedef Elem<T> E;
  constexpr int kOwn = kTile / NW;  // steps of a tile that a wave prepares
  Args p = args();
  const int n0 = at.wave * P, live = PAD ? min(max(p->N - n0, 0), P) : P;
  float A2[P], h[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int n = n0 + i;
    const bool some = at.ok && n < p->N;
    A2[i] = some ? rate(p->A[(int64_t)at.ch * p->N + n]) : 0.0f;
    h[i] = 0.0f;
    if (OUT && some) {
      if (at.chunk) h[i] = p->ends[(((int64_t)(at.chunk - 1) * p->B + at.b) * p->N + n) * p->H + at.ch];
      else if (p->h0 != nullptr) h[i] = p->h0[((int64_t)at.b * p->H + at.ch) * p->N + n];
    }
  }
  const float bias = p->bias != nullptr && at.ok ? p->bias[at.ch] : 0.0f;
  const float D = OUT && p->D != nullptr && at.ok ? p->D[at.ch] : 0.0f;
  const uint32_t off = lane_off<T>(at);
  float span = 0.0f, most = 0.0f;
  bool drop = false;
  unsigned int rd[kOwn], ru[kOwn], rz[kOwn];
  Tile<T, P, NW> tile;
  bool flag;
  auto fetch = [&](int t0) __attribute__((always_inline)) {
    tile.load(p, at, t0);
    flag = load_flag(p, at, t0);
    const int t = t0 + at.wave;
    const T* d = row_of<T>(p->delta, p->sdl_t, p->sdl_b, t, at.b);
    const T* u = row_of<T>(p->u, p->su_t, p->su_b, t, at.b);
    const T* z = row_of<T>(p->z, p->sz_t, p->sz_b, t, at.b);
    const bool gated = OUT && p->z != nullptr;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const uint32_t o = t + NW * i < at.t1 ? off : kOffNone;
      rd[i] = E::load(d + i * NW * p->sdl_t, o);
      ru[i] = E::load(u + i * NW * p->su_t, o);
      if (OUT) rz[i] = E::load(z + i * NW * p->sz_t, gated ? o : kOffNone);
    }
  };
  fetch(at.t0);
  for (int t0 = at.t0; t0 < at.t1; t0 += kTile) {
    float u[kOwn], z[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int s = at.wave + NW * i;
      u[i] = E::value(ru[i]);
      if (OUT) z[i] = E::value(rz[i]);
      const float dt = t0 + s < at.t1 ? softplus(E::value(rd[i]) + bias) : 0.0f;
      lds.xs[s][at.lane] = float2{dt, dt * u[i]};
    }
    tile.put(at, lds.bc);
    const uint32_t flags = mask_of(flag);
    share_barrier();
    if (t0 + kTile < at.t1) fetch(t0 + kTile);
    if (OUT) {
      if (p->saved != nullptr && at.ok) {
        float* to = p->saved + (((int64_t)(t0 / kTile) * p->B + at.b) * p->N + n0) * p->H + at.ch;
#pragma unroll
        for (int i = 0; i < P; ++i)
          if (!PAD || i < live) to[(int64_t)i * p->H] = h[i];
      }
    }
    with_flags(flags, [&](auto F) __attribute__((always_inline)) {
      constexpr bool RESET = decltype(F)::value;
#pragma unroll
      for (int s = 0; s < kTile; ++s) {
        const float2 x = lds.xs[s][at.lane];
        float bm[P], cm[P];
        lds.bc[s][at.wave].read(bm, cm);
        const bool start = RESET && (flags >> s & 1);
        float y = 0.0f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          if (PAD && i >= live) continue;
          if (start) h[i] = 0.0f;
          h[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(x.x * A2[i]), h[i], x.y * bm[i]);
          if (OUT) y = __builtin_fmaf(cm[i], h[i], y);
        }
        if constexpr (OUT) {
          lds.part[at.wave][s][at.lane] = y;
        } else {
          span += x.x;
          most = __builtin_fmaxf(most, x.x);
        }
      }
    });
    if (!OUT && flags) drop = true;
    share_barrier();
    if constexpr (OUT) {
      T* to = row_of<T>(p->y, p->sy_t, p->sy_b, t0 + at.wave, at.b);
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int s = at.wave + NW * i;
        float y = lds.part[0][s][at.lane];
#pragma unroll
        for (int w = 1; w < NW; ++w)
          if (!PAD || w * P < p->N) y += lds.part[w][s][at.lane];
        y = __builtin_fmaf(D, u[i], y);
        if (p->ungated != nullptr)
          Elem<float>::store(row_of<float>(p->ungated, (int64_t)p->B * p->H, p->H, t0 + s, at.b),
                             t0 + s < at.t1 ? lane_off<float>(at) : kOffNone, y);
        const float gate = z[i] * sigmoid(z[i]);
        y = p->z != nullptr ? y * gate : y;
        E::store(to + i * NW * p->sy_t, t0 + s < at.t1 ? off : kOffNone, y);
      }
    }
  }
  if (!at.ok) return;
  const int64_t row = (int64_t)at.chunk * p->B + at.b;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int n = n0 + i;
    if (n >= p->N) continue;
    // what follows a chunk needs its end: the last one's is h_T, the first one's the state itself
    if (OUT && p->h_last != nullptr && at.chunk == p->chunks - 1) p->h_last[((int64_t)at.b * p->H + at.ch) * p->N + n] = h[i];
    if (!OUT || (at.chunk == 0 && p->chunks > 1)) p->ends[(row * p->N + n) * p->H + at.ch] = h[i];
  }
  if (!OUT) {
    if (at.wave == 0) put_span(p, row * p->H + at.ch, drop ? -1.0f : span, most);
  }
}

template <typename T, int P, int NW, bool PAD, bool FIRST>
__global__ __launch_bounds__(64 * NW) void ssm_fwd_kernel(SsmParams p) {
  __shared__ FwdShared<P, NW> lds;
  const At at(p, !FIRST && p.chunks > 1 ? 1 : 0, p.length);
  if (FIRST && at.chunk > 0) fwd_chunk<T, P, NW, PAD, false>(at, lds);
  else fwd_chunk<T, P, NW, PAD, true>(at, lds);
}

// Where waves are many without that, one has 64 channels with all their states to itself, which nothing has to
// be shared for: B and C come from LDS, the same for all lanes.
constexpr int kGroup = 4;  // steps whose loads are in flight together

// A group's B and C on their way to LDS as floats, [step][B, C][NP] with kEach of them a lane side by side.
template <typename T, int NP>
struct Rows {
  static constexpr int kEach = kGroup * 2 * NP >= 64 ? kGroup * 2 * NP / 64 : 1, kLanes = 2 * NP / kEach;  // kLanes a step
  static_assert(NP % kEach == 0, "a lane's elements are of one row");
  const T* at_row;  // of the group that is loaded next
  int64_t by;       // to the group after it
  int step, some;   // the lane's step of a group, and how many of its states exist
  unsigned int x[kEach];
  // groups from t0 on, or back
  __device__ __forceinline__ void init(Args p, const At& at, int t0, bool back) {
    step = at.lane / kLanes;
    const int e = at.lane % kLanes * kEach, n = e % NP;
    const bool c = e >= NP;
    const int64_t st = c ? p->sc_t : p->sb_t;
    at_row = static_cast<const T*>(c ? p->cm : p->bm) + (t0 + step) * st + at.b * (c ? p->sc_b : p->sb_b) + n;
    by = (back ? -kGroup : kGroup) * st;
    some = step < kGroup ? p->N - n : 0;
  }
  __device__ __forceinline__ void load(const At& at, int t0) {
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      x[k] = 0;
      if (t0 + step < at.t1 && k < some) x[k] = sizeof(T) == 2 ? *reinterpret_cast<const unsigned short*>(at_row + k)
                                                               : *reinterpret_cast<const unsigned int*>(at_row + k);
    }
    at_row += by;
  }
  __device__ __forceinline__ void put(float (*lds)[2 * NP], const At& at) const {
#pragma unroll
    for (int k = 0; k < kEach; ++k)
      if (kGroup * kLanes == 64 || at.lane < kGroup * kLanes) (&lds[0][0])[at.lane * kEach + k] = Elem<T>::value(x[k]);
  }
};
// The same NP floats of LDS in every lane.
template <int NP>
__device__ __forceinline__ void read_row(const float* lds, float (&x)[NP]) {
#pragma unroll
  for (int n = 0; n < NP; n += 4) {
    const f4v q = *reinterpret_cast<const f4v*>(lds + n);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[n + k] = q[k];
  }
}

// A wave scans 64 channels, a lane each with all its states, over a chunk. OUT: the scan itself. Otherwise what
// the chunk makes of a zero state, and its sum of dt. PAD: N is less than NP; states that do
// not exist are left out.
template <typename T, int NP, bool PAD, bool OUT>
__device__ __forceinline__ void wide_fwd_chunk(const At& at, float (*bc)[2 * NP]) {
  typedef Elem<T> E;
  Args p = args();
  const int N = PAD ? p->N : NP;
  float A2[NP], h[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    const bool some = at.ok && n < N;
    A2[n] = some ? rate(p->A[(int64_t)at.ch * N + n]) : 0.0f;
    h[n] = 0.0f;
    if (OUT && some) {
      if (at.chunk) h[n] = p->ends[(((int64_t)(at.chunk - 1) * p->B + at.b) * N + n) * p->H + at.ch];
      else if (p->h0 != nullptr) h[n] = p->h0[((int64_t)at.b * p->H + at.ch) * N + n];
    }
  }
  const float bias = p->bias != nullptr && at.ok ? p->bias[at.ch] : 0.0f;
  const float D = OUT && p->D != nullptr && at.ok ? p->D[at.ch] : 0.0f;
  const uint32_t off = lane_off<T>(at);
  const bool gated = OUT && p->z != nullptr, keep = OUT && p->ungated != nullptr;
  float span = 0.0f, most = 0.0f;
  bool drop = false;
  unsigned int rd[kGroup], ru[kGroup], rz[kGroup];
  Rows<T, NP> rows;
  bool flag;
  auto fetch = [&](int t) __attribute__((always_inline)) {
    rows.load(at, t);
    flag = load_flag(p, at, t);
    const T* d = row_of<T>(p->delta, p->sdl_t, p->sdl_b, t, at.b);
    const T* u = row_of<T>(p->u, p->su_t, p->su_b, t, at.b);
    const T* z = row_of<T>(p->z, p->sz_t, p->sz_b, t, at.b);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const uint32_t o = t + i < at.t1 ? off : kOffNone;
      rd[i] = E::load(d + i * p->sdl_t, o);
      ru[i] = E::load(u + i * p->su_t, o);
      if (OUT) rz[i] = E::load(z + i * p->sz_t, gated ? o : kOffNone);
    }
  };
  rows.init(p, at, at.t0, false);
  fetch(at.t0);
  for (int t0 = at.t0; t0 < at.t1; t0 += kGroup) {
    const uint32_t flags = mask_of(flag);
    if (OUT && p->saved != nullptr && t0 % kTile == 0 && at.ok) {
      float* to = p->saved + ((int64_t)(t0 / kTile) * p->B + at.b) * N * p->H + at.ch;
#pragma unroll
      for (int n = 0; n < NP; ++n)
        if (n < N) to[(int64_t)n * p->H] = h[n];
    }
    share_in_wave();
    rows.put(bc, at);
    share_in_wave();
    float dt[kGroup], u[kGroup], z[kGroup];
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      dt[i] = t0 + i < at.t1 ? softplus(E::value(rd[i]) + bias) : 0.0f;
      u[i] = E::value(ru[i]);
      if (OUT) z[i] = E::value(rz[i]);
    }
    if (t0 + kGroup < at.t1) fetch(t0 + kGroup);
    T* to = OUT ? row_of<T>(p->y, p->sy_t, p->sy_b, t0, at.b) : nullptr;
    float* to_u = keep ? row_of<float>(p->ungated, (int64_t)p->B * p->H, p->H, t0, at.b) : nullptr;
    if (!OUT && (flags & ((1u << kGroup) - 1))) drop = true;
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      float bm[NP], cm[NP];
      read_row<NP>(bc[i], bm);
      if (OUT) read_row<NP>(bc[i] + NP, cm);
      const float du = dt[i] * u[i];
      if (flags >> i & 1) {  // uniform
#pragma unroll
        for (int n = 0; n < NP; ++n) h[n] = 0.0f;
      }
      float y = 0.0f;
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        if (PAD && n >= N) continue;
        h[n] = __builtin_fmaf(__builtin_amdgcn_exp2f(dt[i] * A2[n]), h[n], du * bm[n]);
        if (OUT) y = __builtin_fmaf(cm[n], h[n], y);
      }
      if constexpr (OUT) {
        y = __builtin_fmaf(D, u[i], y);
        if (keep) Elem<float>::store(to_u + (int64_t)i * p->B * p->H, t0 + i < at.t1 ? lane_off<float>(at) : kOffNone, y);
        const float gate = z[i] * sigmoid(z[i]);
        E::store(to + i * p->sy_t, t0 + i < at.t1 ? off : kOffNone, gated ? y * gate : y);
      } else {
        span += dt[i];
        most = __builtin_fmaxf(most, dt[i]);
      }
      if (i % 2) __builtin_amdgcn_sched_barrier(0);  // rows of few steps ahead: registers are short
    }
  }
  if (!at.ok) return;
  const int64_t row = (int64_t)at.chunk * p->B + at.b;
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    if (n >= N) continue;
    // what follows a chunk needs its end: the last one's is h_T, the first one's the state itself
    if (OUT && p->h_last != nullptr && at.chunk == p->chunks - 1) p->h_last[((int64_t)at.b * p->H + at.ch) * N + n] = h[n];
    if (!OUT || (at.chunk == 0 && p->chunks > 1)) p->ends[(row * N + n) * p->H + at.ch] = h[n];
  }
  if (!OUT) {
    put_span(p, row * p->H + at.ch, drop ? -1.0f : span, most);
  }
}

template <typename T, int NP, bool PAD, bool FIRST>
__global__ __launch_bounds__(64) void ssm_fwd_wide_kernel(SsmParams p) {
  __shared__ alignas(16) float bc[kGroup][2 * NP];
  const At at(p, !FIRST && p.chunks > 1 ? 1 : 0, p.length);
  if (FIRST && at.chunk > 0) wide_fwd_chunk<T, NP, PAD, false>(at, bc);
  else wide_fwd_chunk<T, NP, PAD, true>(at, bc);
}

// What becomes of a state s, or of a gradient on its way back, over steps whose sizes are `over` in sum and `most` at
// the largest, as a step at a time gives it, where exp2(A2 over) s does not say it: of an infinite one something is left
// unless a step alone leaves nothing (0 x infinity), and growth past float32's range (a rate above 0) may be of one that does not
// get there.
constexpr float kUnusual = 1.0e38f;  // so where a state, or what is left of one, is as large or larger
__device__ __forceinline__ float passed(float s, float A2, float over, float most) {
  if (s == 0.0f || __builtin_fabsf(s) == __builtin_inff()) return s * __builtin_amdgcn_exp2f(A2 * most);
  const float v = __builtin_fminf(__builtin_fmaxf(A2 * over, -1000.0f), 1000.0f), e = __builtin_rintf(v);
  return __builtin_ldexpf(s * __builtin_amdgcn_exp2f(v - e), (int)e);
}

// Forward: the states at the chunks' ends. Slot 0 of `ends` holds that of the first chunk, slot c what
// chunk c makes of zero, and on return the state after it. BACK: slot c holds what part c of the axis
// sends back of a zero gradient, and on return of the whole: from the last part to the second chunk's first.
template <bool BACK>
__global__ __launch_bounds__(64) void ssm_join_kernel(SsmParams p) {
  constexpr int kAhead = 16;  // slots whose loads are in flight together
  const int64_t plane = (int64_t)p.B * p.N * p.H, e = (int64_t)blockIdx.x * 64 + threadIdx.x;
  if (e >= plane) return;
  const int ch = (int)(e % p.H), n = (int)(e / p.H % p.N), b = (int)(e / p.H / p.N);
  const float A2 = rate(p.A[(int64_t)ch * p.N + n]);
  float s = 0.0f;
  if (!BACK) s = p.ends[e];
  if (BACK && p.dh_last != nullptr) s = p.dh_last[((int64_t)b * p.H + ch) * p.N + n];
  const int all = parts_of(p), count = BACK ? all - p.each : p.chunks - 2, first = BACK ? all - 1 : 1;
  const int64_t step = BACK ? -plane : plane, span_step = (BACK ? -1 : 1) * (int64_t)p.B * p.H;
  float* slot = p.ends + first * plane + e;
  const float* span = p.span + ((int64_t)first * p.B + b) * p.H + ch;
  const int64_t most = (int64_t)p.chunks * p.each * p.B * p.H;  // from a sum to the largest
  for (int k0 = 0; k0 < count; k0 += kAhead) {
    float end[kAhead], over[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      end[k] = over[k] = 0.0f;
      if (k0 + k >= count) continue;  // uniform
      end[k] = slot[k * step];
      over[k] = span[k * span_step];
    }
    const float before = s;
    float largest = 0.0f;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (k0 + k >= count) continue;
      const float decay = __builtin_amdgcn_exp2f(A2 * over[k]);
      const bool drop = over[k] < 0.0f;
      largest = __builtin_fmaxf(__builtin_fmaxf(largest, __builtin_fabsf(s)), decay);
      s = drop ? end[k] : __builtin_fmaf(decay, s, end[k]);
      slot[k * step] = s;
    }
    if (__builtin_amdgcn_ballot_w64(largest >= kUnusual)) {  // uniform, and seldom: these slots again
      s = before;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (k0 + k >= count) continue;
        const float decay = __builtin_amdgcn_exp2f(A2 * over[k]);
        if (over[k] < 0.0f) s = end[k];
        else if (__builtin_fmaxf(__builtin_fabsf(s), decay) >= kUnusual) s = passed(s, A2, over[k], span[k * span_step + most]) + end[k];
        else s = __builtin_fmaf(decay, s, end[k]);  // as above: a lane's result is its own
        slot[k * step] = s;
      }
    }
    slot += kAhead * step;
    span += kAhead * span_step;
  }
}

template <int P, int NW>
struct BwdShared {
  float2 xs[kTile][64];  // dt, dt u
  float ds[kTile][64];   // dy
  // [1] stays zero: what lanes without a channel read, so that sums over lanes do not see them
  Pair<P> bc[2][kTile][NW];
  // A step's decays of the wave's states, left for the way back, and then, in the first two of their
  // places, the wave's parts of S and of sum_n q A / ln 2.
  struct alignas(4 * P) Step {
    float x[P];
  } part[NW][kTile][64];
};

// The gradient that a chunk sends to the state before it, from a zero gradient after it.
template <typename T, int P, int NW, bool PAD>
__global__ __launch_bounds__(64 * NW) void ssm_bwd_ends_kernel(SsmParams kernel_args) {
  __shared__ float2 xs[kTile][64];  // dt, dy
  __shared__ Pair<P> bc[kTile][NW];
  typedef Elem<T> E;
  constexpr int kOwn = kTile / NW;
  const At at(kernel_args, 1, kernel_args.length);
  Args p = args();
  const int n0 = at.wave * P, live = PAD ? min(max(p->N - n0, 0), P) : P;
  float A2[P], e[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    A2[i] = at.ok && n0 + i < p->N ? rate(p->A[(int64_t)at.ch * p->N + n0 + i]) : 0.0f;
    e[i] = 0.0f;
  }
  const float bias = p->bias != nullptr && at.ok ? p->bias[at.ch] : 0.0f;
  const uint32_t off = lane_off<T>(at);
  float span = 0.0f, most = 0.0f;
  bool drop = false;
  unsigned int rd[kOwn], rz[kOwn], rg[kOwn];
  Tile<T, P, NW> tile;
  bool flag;
  auto fetch = [&](int t0) __attribute__((always_inline)) {
    tile.load(p, at, t0);
    flag = load_flag(p, at, t0);
    const int t = t0 + at.wave;
    const T* d = row_of<T>(p->delta, p->sdl_t, p->sdl_b, t, at.b);
    const T* g = row_of<T>(p->dy, p->sdy_t, p->sdy_b, t, at.b);
    const T* z = row_of<T>(p->z, p->sz_t, p->sz_b, t, at.b);
    const bool gated = p->z != nullptr;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const uint32_t o = t + NW * i < at.t1 ? off : kOffNone;
      rd[i] = E::load(d + i * NW * p->sdl_t, o);
      rg[i] = E::load(g + i * NW * p->sdy_t, o);
      rz[i] = E::load(z + i * NW * p->sz_t, gated ? o : kOffNone);
    }
  };
  const int last = at.t0 + (at.t1 - at.t0 - 1) / kTile * kTile;
  fetch(last);
  for (int t0 = last; t0 >= at.t0; t0 -= kTile) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int s = at.wave + NW * i;
      const float dt = t0 + s < at.t1 ? softplus(E::value(rd[i]) + bias) : 0.0f;
      const float z = E::value(rz[i]), g = E::value(rg[i]);
      xs[s][at.lane] = float2{dt, p->z != nullptr ? g * (z * sigmoid(z)) : g};
    }
    tile.put(at, bc);
    const uint32_t flags = mask_of(flag);
    share_barrier();
    if (t0 > at.t0) fetch(t0 - kTile);
    with_flags(flags, [&](auto F) __attribute__((always_inline)) {
      constexpr bool RESET = decltype(F)::value;
#pragma unroll
      for (int s = kTile - 1; s >= 0; --s) {
        const float2 x = xs[s][at.lane];
        float bm[P], cm[P];
        bc[s][at.wave].read(bm, cm);
#pragma unroll
        for (int i = 0; i < P; ++i) {
          if (PAD && i >= live) continue;
          e[i] = __builtin_amdgcn_exp2f(x.x * A2[i]) * __builtin_fmaf(cm[i], x.y, e[i]);
          if (RESET && (flags >> s & 1)) e[i] = 0.0f;
        }
        span += x.x;
        most = __builtin_fmaxf(most, x.x);
      }
    });
    if (flags) drop = true;
    share_barrier();
  }
  if (!at.ok) return;
  const int64_t row = (int64_t)at.chunk * p->B + at.b;
#pragma unroll
  for (int i = 0; i < P; ++i)
    if (n0 + i < p->N) p->ends[(row * p->N + n0 + i) * p->H + at.ch] = e[i];
  if (at.wave == 0) put_span(p, row * p->H + at.ch, drop ? -1.0f : span, most);
}

// The gradient that a part of the axis sends to the state before it, from a zero gradient after
// it, and its sum of dt. A wave takes 64 channels, as forwards.
template <typename T, int NP, bool PAD>
__global__ __launch_bounds__(64) void ssm_bwd_ends_wide_kernel(SsmParams) {
  typedef Elem<T> E;
  __shared__ alignas(16) float bc[kGroup][2 * NP];
  Args p = args();
  SsmParams q;
  q.blocks = p->blocks;
  q.B = p->B;
  q.H = p->H;
  q.T = p->T;
  const At at(q, p->each, p->length / p->each);
  const int N = PAD ? p->N : NP;
  float A2[NP], e[NP];
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    A2[n] = at.ok && n < N ? rate(p->A[(int64_t)at.ch * N + n]) : 0.0f;
    e[n] = 0.0f;
  }
  const float bias = p->bias != nullptr && at.ok ? p->bias[at.ch] : 0.0f;
  const uint32_t off = lane_off<T>(at);
  const bool gated = p->z != nullptr;
  float span = 0.0f, most = 0.0f;
  bool drop = false;
  unsigned int rd[kGroup], rz[kGroup], rg[kGroup];
  Rows<T, NP> rows;
  bool flag;
  auto fetch = [&](int t) __attribute__((always_inline)) {
    rows.load(at, t);
    flag = load_flag(p, at, t);
    const T* d = row_of<T>(p->delta, p->sdl_t, p->sdl_b, t, at.b);
    const T* g = row_of<T>(p->dy, p->sdy_t, p->sdy_b, t, at.b);
    const T* z = row_of<T>(p->z, p->sz_t, p->sz_b, t, at.b);
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const uint32_t o = t + i < at.t1 ? off : kOffNone;
      rd[i] = E::load(d + i * p->sdl_t, o);
      rg[i] = E::load(g + i * p->sdy_t, o);
      rz[i] = E::load(z + i * p->sz_t, gated ? o : kOffNone);
    }
  };
  const int last = at.t0 + (at.t1 - at.t0 - 1) / kGroup * kGroup;
  rows.init(p, at, last, true);
  fetch(last);
  for (int t0 = last; t0 >= at.t0; t0 -= kGroup) {
    const uint32_t flags = mask_of(flag);
    share_in_wave();
    rows.put(bc, at);
    share_in_wave();
    float dt[kGroup], dy[kGroup];
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      dt[i] = t0 + i < at.t1 ? softplus(E::value(rd[i]) + bias) : 0.0f;
      const float z = E::value(rz[i]), g = E::value(rg[i]);
      dy[i] = gated ? g * (z * sigmoid(z)) : g;
    }
    if (t0 > at.t0) fetch(t0 - kGroup);
    if (flags & ((1u << kGroup) - 1)) drop = true;
#pragma unroll
    for (int i = kGroup - 1; i >= 0; --i) {
      float cm[NP];
      read_row<NP>(bc[i] + NP, cm);
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        if (PAD && n >= N) continue;
        e[n] = __builtin_amdgcn_exp2f(dt[i] * A2[n]) * __builtin_fmaf(cm[n], dy[i], e[n]);
      }
      if (flags >> i & 1) {  // uniform
#pragma unroll
        for (int n = 0; n < NP; ++n) e[n] = 0.0f;
      }
      span += dt[i];
      most = __builtin_fmaxf(most, dt[i]);
    }
  }
  if (!at.ok) return;
  const int64_t row = (int64_t)at.chunk * p->B + at.b;
#pragma unroll
  for (int n = 0; n < NP; ++n)
    if (n < N) p->ends[(row * N + n) * p->H + at.ch] = e[n];
  put_span(p, row * p->H + at.ch, drop ? -1.0f : span, most);
}

template <typename T, int P, int NW, bool PAD>
__device__ __forceinline__ void bwd_chunk(At at, BwdShared<P, NW>& lds) {
  typedef Elem<T> E;
  constexpr int kOwn = kTile / NW;
  Args p = args();
  const int n0 = at.wave * P, live = PAD ? min(max(p->N - n0, 0), P) : P;
  float A2[P], e[P], dA[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int n = n0 + i;
    const bool some = at.ok && n < p->N;
    A2[i] = some ? rate(p->A[(int64_t)at.ch * p->N + n]) : 0.0f;
    dA[i] = 0.0f;
    e[i] = 0.0f;
    if (some) {
      if (at.chunk < p->chunks - 1) e[i] = p->ends[(((int64_t)(at.chunk + 1) * p->each * p->B + at.b) * p->N + n) * p->H + at.ch];
      else if (p->dh_last != nullptr) e[i] = p->dh_last[((int64_t)at.b * p->H + at.ch) * p->N + n];
    }
  }
  const float bias = p->bias != nullptr && at.ok ? p->bias[at.ch] : 0.0f;
  const float D = p->D != nullptr && at.ok ? p->D[at.ch] : 0.0f;
  const uint32_t off = lane_off<T>(at);
  float dD = 0.0f, dbias = 0.0f;
  for (int i = threadIdx.x; i < kTile * NW * 2 * P; i += 64 * NW) (&lds.bc[1][0][0].x[0])[i] = 0.0f;
  unsigned int rd[kOwn], ru[kOwn], rz[kOwn], rg[kOwn], ry[kOwn];
  auto fetch = [&](int t0) __attribute__((always_inline)) {
    Args p = args();
    const int t = t0 + at.wave;
    const T* d = row_of<T>(p->delta, p->sdl_t, p->sdl_b, t, at.b);
    const T* u = row_of<T>(p->u, p->su_t, p->su_b, t, at.b);
    const T* g = row_of<T>(p->dy, p->sdy_t, p->sdy_b, t, at.b);
    const T* z = row_of<T>(p->z, p->sz_t, p->sz_b, t, at.b);
    const float* y = row_of<float>(p->ungated, (int64_t)p->B * p->H, p->H, t, at.b);
    const bool gated = p->z != nullptr;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const bool some = t + NW * i < at.t1;
      const uint32_t o = some ? off : kOffNone;
      rd[i] = E::load(d + i * NW * p->sdl_t, o);
      ru[i] = E::load(u + i * NW * p->su_t, o);
      rg[i] = E::load(g + i * NW * p->sdy_t, o);
      rz[i] = E::load(z + i * NW * p->sz_t, gated ? o : kOffNone);
      ry[i] = Elem<float>::load(y + (int64_t)i * NW * p->B * p->H, gated && some ? lane_off<float>(at) : kOffNone);
    }
  };
  const int last = at.t0 + (at.t1 - at.t0 - 1) / kTile * kTile;
  fetch(last);
  for (int t0 = last; t0 >= at.t0; t0 -= kTile) {
    p = args();
    asm volatile("" : "+v"(at.lane), "+s"(at.wave));  // addresses made from these are made anew, not kept
    const Pair<P>(*const bc)[NW] = lds.bc[at.ok ? 0 : 1];
    const bool gated = p->z != nullptr;
    // loaded a tile ahead, these would take registers that are not there
    Tile<T, P, NW> tile;
    tile.load(p, at, t0);
    const bool flag = load_flag(p, at, t0);
    float start[P];
    const float* from = p->saved + (((int64_t)(t0 / kTile) * p->B + at.b) * p->N + n0) * p->H + at.ch;
#pragma unroll
    for (int i = 0; i < P; ++i) start[i] = at.ok && (!PAD || i < live) ? from[(int64_t)i * p->H] : 0.0f;
    float u[kOwn], x[kOwn];
    T* to_z = row_of<T>(p->dz, p->sdz_t, p->sdz_b, t0 + at.wave, at.b);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int s = at.wave + NW * i;
      u[i] = E::value(ru[i]);
      x[i] = E::value(rd[i]) + bias;
      const float dt = t0 + s < at.t1 ? softplus(x[i]) : 0.0f;
      const float z = E::value(rz[i]), g = sigmoid(z), d = E::value(rg[i]);
      if (gated)
        E::store(to_z + i * NW * p->sdz_t, t0 + s < at.t1 ? off : kOffNone,
                 d * g * __builtin_fmaf(z, 1.0f - g, 1.0f) * Elem<float>::value(ry[i]));
      lds.xs[s][at.lane] = float2{dt, dt * u[i]};
      lds.ds[s][at.lane] = gated ? d * (z * g) : d;
    }
    tile.put(at, lds.bc[0]);
    const uint32_t flags = mask_of(flag);
    share_barrier();
    with_flags(flags, [&](auto F) __attribute__((always_inline)) {
      constexpr bool RESET = decltype(F)::value;
      // after each step
      float h[kTile][P];
#pragma unroll
      for (int s = 0; s < kTile; ++s) {
        const float2 v = lds.xs[s][at.lane];
        float bm[P], cm[P];
        bc[s][at.wave].read(bm, cm);
        typename BwdShared<P, NW>::Step decay;
#pragma unroll
        for (int i = 0; i < P; ++i) {
          h[s][i] = decay.x[i] = 0.0f;
          if (PAD && i >= live) continue;
          float before = s ? h[s > 0 ? s - 1 : 0][i] : start[i];
          if (RESET && (flags >> s & 1)) before = 0.0f;
          decay.x[i] = __builtin_amdgcn_exp2f(v.x * A2[i]);
          h[s][i] = __builtin_fmaf(decay.x[i], before, v.y * bm[i]);
        }
        lds.part[at.wave][s][at.lane] = decay;
        if (s % 2) __builtin_amdgcn_sched_barrier(0);  // loads of few steps ahead: registers are short
      }
      uint32_t back = flags;
      asm volatile("" : "+s"(back));  // what a reset drops is found anew, not kept
      __builtin_amdgcn_sched_barrier(0);
      // back over the tile; sums over the lanes of dB and dC of a pair of states in one register a step
      float sums[P / 2][kTile];
#pragma unroll
      for (int s = kTile - 1; s >= 0; --s) {
        const float2 v = lds.xs[s][at.lane];
        const float g = lds.ds[s][at.lane];
        float bm[P], cm[P], S = 0.0f, Q = 0.0f, db[P], dc[P];
        bc[s][at.wave].read(bm, cm);
        const typename BwdShared<P, NW>::Step decay = lds.part[at.wave][s][at.lane];
#pragma unroll
        for (int i = 0; i < P; ++i) {
          db[i] = dc[i] = 0.0f;
          if (PAD && i >= live) continue;
          const float G = __builtin_fmaf(cm[i], g, e[i]);
          float before = s ? h[s > 0 ? s - 1 : 0][i] : start[i];
          e[i] = decay.x[i] * G;
          if (RESET && (back >> s & 1)) e[i] = before = 0.0f;
          const float q = e[i] * before;
          S = __builtin_fmaf(G, bm[i], S);
          Q = __builtin_fmaf(q, A2[i], Q);
          dA[i] = __builtin_fmaf(q, v.x, dA[i]);
          db[i] = G * v.y;
          dc[i] = h[s][i] * g;
        }
        lds.part[at.wave][s][at.lane].x[0] = S;
        lds.part[at.wave][s][at.lane].x[1] = Q;
#pragma unroll
        for (int i = 0; i < P; i += 2)
          sums[i / 2][s] = join<16>(join<32>(db[i], db[i + 1]), join<32>(dc[i], dc[i + 1]));
        if (s == kTile / 2 && t0 > at.t0) fetch(t0 - kTile);  // half of h is done with
        __builtin_amdgcn_sched_barrier(0);
      }
      Args p = args();
#pragma unroll
      for (int k = 0; k < P / 2; ++k) {
        float w8[8], w4[4], w2[2];
#pragma unroll
        for (int s = 0; s < 8; ++s) w8[s] = join<1>(sums[k][2 * s], sums[k][2 * s + 1]);
#pragma unroll
        for (int s = 0; s < 4; ++s) w4[s] = join<2>(w8[2 * s], w8[2 * s + 1]);
#pragma unroll
        for (int s = 0; s < 2; ++s) w2[s] = join<4>(w4[2 * s], w4[2 * s + 1]);
        const float sum = join<8>(w2[0], w2[1]);
        const int t = t0 + (at.lane & 15), n = n0 + 2 * k + (at.lane >> 5);
        if (t < at.t1 && n < p->N)
          p->part_bc[(((int64_t)at.block * p->T + t) * p->B + at.b) * 2 * p->N + (at.lane & 16 ? p->N : 0) + n] = sum;
      }
    });
    share_barrier();
    p = args();
    T* to_u = row_of<T>(p->du, p->sdu_t, p->sdu_b, t0 + at.wave, at.b);
    T* to_d = row_of<T>(p->ddelta, p->sdd_t, p->sdd_b, t0 + at.wave, at.b);
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int s = at.wave + NW * i;
      float2 v{lds.part[0][s][at.lane].x[0], lds.part[0][s][at.lane].x[1]};
#pragma unroll
      for (int w = 1; w < NW; ++w)
        if (!PAD || w * P < p->N) {
          v.x += lds.part[w][s][at.lane].x[0];
          v.y += lds.part[w][s][at.lane].x[1];
        }
      const float dt = lds.xs[s][at.lane].x, dy = lds.ds[s][at.lane];
      const float dd = __builtin_fmaf(u[i], v.x, v.y * kLn2) * sigmoid(x[i]);
      const uint32_t o = t0 + s < at.t1 ? off : kOffNone;
      E::store(to_u + i * NW * p->sdu_t, o, __builtin_fmaf(dt, v.x, D * dy));
      E::store(to_d + i * NW * p->sdd_t, o, dd);
      if (t0 + s < at.t1) {
        dD = __builtin_fmaf(u[i], dy, dD);
        dbias += dd;
      }
    }
  }
  // sums over the chunk: dA of the wave's states, dD and dbias over the waves
  p = args();
  const int64_t row = (int64_t)at.chunk * p->B + at.b, parts = row * (p->N + 2);
  if (at.ok) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      const int n = n0 + i;
      if (n >= p->N) continue;
      p->part_a[(parts + n) * p->H + at.ch] = dA[i];
      if (at.chunk == 0 && p->dh0 != nullptr) p->dh0[((int64_t)at.b * p->H + at.ch) * p->N + n] = e[i];
    }
  }
  share_barrier();
  lds.part[at.wave][0][at.lane].x[0] = dD;
  lds.part[at.wave][0][at.lane].x[1] = dbias;
  share_barrier();
  if (at.wave == 0 && at.ok) {
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      dD += lds.part[w][0][at.lane].x[0];
      dbias += lds.part[w][0][at.lane].x[1];
    }
    p->part_a[(parts + p->N) * p->H + at.ch] = dD;
    p->part_a[(parts + p->N + 1) * p->H + at.ch] = dbias;
  }
}

template <typename T, int P, int NW, bool PAD>
__global__ __launch_bounds__(64 * NW, P == 2 && NW == 8 ? 4 : 2) void ssm_bwd_kernel(SsmParams p) {
  __shared__ BwdShared<P, NW> lds;
  bwd_chunk<T, P, NW, PAD>(At(p, 0, p.length), lds);
}

// What the workgroups' sums make together, in order: dB and dC [T, B, N] over the channel blocks, by the first
// bc_groups workgroups; dA [H, N], dD and dbias [H] over chunks and batch rows by the others, whose lanes are channels
// and whose four waves take every fourth part.
struct SumParams {
  const float *part_bc, *part_a;
  void *dbm, *dcm;
  float *dA, *dD, *dbias;
  int64_t rows;  // T B
  int H, N, blocks, parts, bc_groups;
};

template <typename T>
__device__ __forceinline__ void sum_bc(const SumParams& p) {
  const int64_t plane = p.rows * 2 * p.N;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < plane; e += (int64_t)p.bc_groups * 256) {
    float s = 0.0f;
    for (int k0 = 0; k0 < p.blocks; k0 += 8) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = k0 + k < p.blocks ? p.part_bc[(k0 + k) * plane + e] : 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k0 + k < p.blocks) s += x[k];
    }
    const int64_t row = e / (2 * p.N);
    const int n = (int)(e - row * 2 * p.N);
    void* dst = n < p.N ? p.dbm : p.dcm;
    if (dst != nullptr) static_cast<T*>(dst)[row * p.N + (n < p.N ? n : n - p.N)] = (T)s;
  }
}

__device__ __forceinline__ void sum_a(const SumParams& p, int group, float (*red)[64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = group / p.blocks, ch = (group - n * p.blocks) * 64 + lane;
  const int64_t plane = (int64_t)(p.N + 2) * p.H;
  const float* src = p.part_a + (int64_t)n * p.H + ch;
  float s = 0.0f;
  if (ch < p.H) {
    for (int k0 = wave; k0 < p.parts; k0 += 4 * 16) {
      float x[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) x[k] = k0 + 4 * k < p.parts ? src[(k0 + 4 * k) * plane] : 0.0f;
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (k0 + 4 * k < p.parts) s += x[k];
    }
  }
  red[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || ch >= p.H) return;
  s = ((s + red[1][lane]) + red[2][lane]) + red[3][lane];
  float* dst = n < p.N ? p.dA : n == p.N ? p.dD : p.dbias;
  if (dst != nullptr) dst[n < p.N ? (int64_t)ch * p.N + n : ch] = s;
}

template <typename T>
__global__ __launch_bounds__(256) void ssm_sum_kernel(SumParams p) {
  __shared__ float red[4][64];
  if ((int)blockIdx.x < p.bc_groups) sum_bc<T>(p);
  else sum_a(p, (int)blockIdx.x - p.bc_groups, red);
}

// One token for each row of a batch of requests, whose states are rows of a cache [S, H, N]:
// four lanes a channel, which hold four states side by side in turn (or, where states are not a multiple of
// four, every fourth one). One launch. B 301, H 1002 in fp32: 15.2 -> 10.8 us with whole accesses, 4 TB/s.
struct SsmStepParams {
  const void *u, *delta, *z, *bm, *cm;
  const float *A, *D, *bias;
  float* state;
  const int32_t* slots;
  void* y;
  int64_t su, sdl, sz, sb, sc, ss, sy;
  int B, H, N, S;
};

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void ssm_step_kernel(SsmStepParams p) {
  const int q = threadIdx.x & 3, ch = blockIdx.x * 64 + (threadIdx.x >> 2), b = blockIdx.y;
  if (ch >= p.H) return;
  const int slot = p.slots ? p.slots[b] : b;
  T* out = static_cast<T*>(p.y) + b * p.sy + ch;
  if (slot < 0 || slot >= p.S) {
    if (q == 0) *out = (T)(slot < 0 ? 0.0f : __builtin_nanf(""));
    return;
  }
  const float u = (float)(static_cast<const T*>(p.u) + b * p.su)[ch];
  const float dt = softplus((float)(static_cast<const T*>(p.delta) + b * p.sdl)[ch] + (p.bias ? p.bias[ch] : 0.0f));
  const T *bm = static_cast<const T*>(p.bm) + b * p.sb, *cm = static_cast<const T*>(p.cm) + b * p.sc;
  const float* A = p.A + (int64_t)ch * p.N;
  float* h = p.state + slot * p.ss + (int64_t)ch * p.N;
  float y = 0.0f;
  auto state = [&](int n, float a, float before) __attribute__((always_inline)) {
    const float x = __builtin_fmaf(__builtin_amdgcn_exp2f(dt * rate(a)), before, dt * u * (float)bm[n]);
    y = __builtin_fmaf((float)cm[n], x, y);
    return x;
  };
  if constexpr (VEC) {
    for (int n = 4 * q; n < p.N; n += 16) {
      const f4v a = *reinterpret_cast<const f4v*>(A + n);
      f4v x = *reinterpret_cast<const f4v*>(h + n);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = state(n + i, a[i], x[i]);
      *reinterpret_cast<f4v*>(h + n) = x;
    }
  } else {
    for (int n = q; n < p.N; n += 4) h[n] = state(n, A[n], h[n]);
  }
  y += lane_xor_c<1>(y);
  y += lane_xor_c<2>(y);
  if (p.D) y = __builtin_fmaf(p.D[ch], u, y);
  if (p.z) {
    const float z = (float)(static_cast<const T*>(p.z) + b * p.sz)[ch];
    y *= z * sigmoid(z);
  }
  if (q == 0) *out = (T)y;
}

// ---- host ---------------------------------------------------------------------------

constexpr int kMostStates = 32;

// Chunks of the time axis, multiples of a tile: workgroups (or, for kernels that share nothing, waves) for every
// CU in each launch. Forwards there are two launches, which have one chunk fewer each; backwards one over
// all chunks, after the waves that find the ends of their parts.
struct Plan {
  int blocks, chunks, length, each;
  bool wide;  // the kernels that share nothing, for the forward or the backward's ends
};
// In us, states over a workgroup's waves / waves that share nothing, the same tensors:
//   T 4096, B 8, H 1024 bf16 training, N 16    912 / 890     T 512, B 16, H 512 fp32 training, N 16   154 / 161
//   the same, N 4                              969 / 700     the same, N 32                           243 / 280
//   the same, N 32                            1665 / 1771    T 1001, B 3, H 333 fp32 training, N 16   140 / 148
//   T 65536, B 1, H 1024 bf16 forward, N 16    627 / 546
// The first with 256, 512 and 1024 workgroups asked for in the backward: N 16 1099, 890, 916; N 32 1758, 1771, 1829; N 4, whose
// workgroups are two waves, 1043, 700, 507. With 2048, 4096 and 8192 waves: N 16 1009, 890, 900. The constants are
// those that are best at N 16; the plan does not ask for N.
constexpr int64_t kGroups = 512;    // workgroups asked for: two a CU (one at a time of N > 16, which fill its LDS)
constexpr int64_t kWaves = 4096;    // waves asked for, where they share nothing
constexpr int64_t kFewWaves = 2048; // up to these, states are spread over the waves of a workgroup
constexpr int kLeastChunk = 64, kLeastPart = 32;  // steps
Plan make_plan(int64_t T, int64_t B, int64_t H, bool back) {
  Plan r;
  r.blocks = (int)((H + 63) / 64);
  const int64_t groups = r.blocks * B, fine = std::max<int64_t>(1, T / kLeastPart), most = std::max<int64_t>(1, T / kLeastChunk);
  auto cut = [](int64_t n, int64_t parts) { return ((n + parts - 1) / parts + kTile - 1) / kTile * kTile; };
  int64_t length;
  r.each = 1;
  r.wide = groups * fine > kFewWaves;
  if (back) {
    const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>(kGroups / groups, most));
    length = cut(T, chunks);
    if (chunks > 1 && r.wide) {
      r.each = (int)std::max<int64_t>(1, std::min<int64_t>(kWaves / (groups * chunks), length / kLeastPart));
      length = cut(length, r.each) * r.each;
    }
  } else {
    int64_t chunks = r.wide ? std::min<int64_t>(1 + kWaves / groups, fine) : std::min<int64_t>(1 + kGroups / groups, most);
    if (chunks < 3) chunks = 1;  // two launches of one chunk each
    length = cut(T, chunks);
  }
  r.length = (int)length;
  r.chunks = (int)((T + length - 1) / length);
  return r;
}

// States that the kernels are made for.
int padded(int64_t N) { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : 32; }

typedef void (*SsmFn)(SsmParams);
enum { kFwd, kFwdFirst, kBwdEnds, kBwd };
template <typename T, int NP, int P, bool PAD>
SsmFn kernel_at(int which, bool wide) {
  switch (which) {
    case kFwd: return wide ? ssm_fwd_wide_kernel<T, NP, PAD, false> : ssm_fwd_kernel<T, P, NP / P, PAD, false>;
    case kFwdFirst: return wide ? ssm_fwd_wide_kernel<T, NP, PAD, true> : ssm_fwd_kernel<T, P, NP / P, PAD, true>;
    case kBwdEnds: return wide ? ssm_bwd_ends_wide_kernel<T, NP, PAD> : ssm_bwd_ends_kernel<T, P, NP / P, PAD>;
    default: return ssm_bwd_kernel<T, P, NP / P, PAD>;
  }
}
template <typename T, int NP, int P>
SsmFn kernel_in(int which, bool wide, int N, int& threads) {
  threads = wide && which != kBwd ? 64 : 64 * NP / P;
  return N == NP ? kernel_at<T, NP, P, false>(which, wide) : kernel_at<T, NP, P, true>(which, wide);
}
template <typename T>
SsmFn kernel_for(int which, bool wide, int N, int& threads) {
  switch (padded(N)) {
    case 4: return kernel_in<T, 4, 2>(which, wide, N, threads);
    case 8: return kernel_in<T, 8, 2>(which, wide, N, threads);
    case 16: return kernel_in<T, 16, 2>(which, wide, N, threads);
    default: return kernel_in<T, 32, 4>(which, wide, N, threads);
  }
}

int launch(int which, bool wide, int dtype, const SsmParams& p, int64_t groups, hipStream_t stream) {
  int threads = 0;
  const SsmFn fn = dtype == GS_DTYPE_F32 ? kernel_for<float>(which, wide, p.N, threads)
                                         : kernel_for<__bf16>(which, wide, p.N, threads);
  hipLaunchKernelGGL(fn, dim3((unsigned)groups), dim3(threads), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}

int check_sizes(const char* who, int64_t T, int64_t B, int64_t H, int64_t N, int dtype) {
  if (T < 1) return set_error(GS_ERR_INVALID, "%s: seq length T must be > 0; got T=%lld", who, (long long)T);
  if (B < 1) return set_error(GS_ERR_INVALID, "%s: batch size B must be > 0; got B=%lld", who, (long long)B);
  if (H < 1) return set_error(GS_ERR_INVALID, "%s: channels H must be > 0; got H=%lld", who, (long long)H);
  if (N < 1 || N > kMostStates)
    return set_error(GS_ERR_INVALID, "%s: states N must be 1 to %d; got N=%lld", who, kMostStates, (long long)N);
  if (T > (1ll << 30) || B > (1ll << 20) || H > (1ll << 20))
    return set_error(GS_ERR_INVALID, "%s: T/B/H out of supported range (T=%lld, B=%lld, H=%lld)", who, (long long)T,
                     (long long)B, (long long)H);
  // workgroups of 512 threads, counted in 32 bits by a launch; chunks only add some where these are few
  if ((H + 63) / 64 * B > (1ll << 22))
    return set_error(GS_ERR_INVALID, "%s: more workgroups than a launch holds (B=%lld, H=%lld)", who, (long long)B, (long long)H);
  return check_dtype(who, dtype);
}

struct Bytes {
  int64_t ends = 0, span = 0, bc = 0, a = 0, total = 0;  // offsets
};
Bytes bytes_of(const Plan& plan, int64_t T, int64_t B, int64_t H, int64_t N, bool back) {
  Bytes r;
  if (plan.chunks > 1) {
    const int64_t parts = (int64_t)plan.chunks * plan.each;
    r.span = align256(parts * B * N * H * 4);
    r.total = r.span + align256(parts * B * H * 8);
  }
  if (back) {
    r.bc = r.total;
    r.a = r.bc + align256(plan.blocks * T * B * 2 * N * 4);
    r.total = r.a + align256(plan.chunks * B * (N + 2) * H * 4);
  }
  return r;
}

int check_fwd(const gs_ssm_args* a, const char* who) {
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  int rc = check_sizes(who, a->T, a->B, a->H, a->N, a->dtype);
  if (rc) return rc;
  if ((rc = check_step_rows(who, "u", a->T, a->B, a->H, a->su_t, a->su_b, false))) return rc;
  if ((rc = check_step_rows(who, "delta", a->T, a->B, a->H, a->sdl_t, a->sdl_b, false))) return rc;
  if ((rc = check_step_rows(who, "z", a->T, a->B, a->H, a->sz_t, a->sz_b, false))) return rc;
  if ((rc = check_step_rows(who, "B", a->T, a->B, a->N, a->sb_t, a->sb_b, false))) return rc;
  if ((rc = check_step_rows(who, "C", a->T, a->B, a->N, a->sc_t, a->sc_b, false))) return rc;
  if ((rc = check_step_rows(who, "reset", a->T, a->B, 1, a->sr_t, a->sr_b, false))) return rc;
  return check_step_rows(who, "y", a->T, a->B, a->H, a->sy_t, a->sy_b, true);
}

int check_bwd(const gs_ssm_bwd_args* a, const char* who) {
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  int rc = check_sizes(who, a->T, a->B, a->H, a->N, a->dtype);
  if (rc) return rc;
  if ((rc = check_step_rows(who, "u", a->T, a->B, a->H, a->su_t, a->su_b, false))) return rc;
  if ((rc = check_step_rows(who, "delta", a->T, a->B, a->H, a->sdl_t, a->sdl_b, false))) return rc;
  if ((rc = check_step_rows(who, "z", a->T, a->B, a->H, a->sz_t, a->sz_b, false))) return rc;
  if ((rc = check_step_rows(who, "B", a->T, a->B, a->N, a->sb_t, a->sb_b, false))) return rc;
  if ((rc = check_step_rows(who, "C", a->T, a->B, a->N, a->sc_t, a->sc_b, false))) return rc;
  if ((rc = check_step_rows(who, "reset", a->T, a->B, 1, a->sr_t, a->sr_b, false))) return rc;
  if ((rc = check_step_rows(who, "dy", a->T, a->B, a->H, a->sdy_t, a->sdy_b, false))) return rc;
  if ((rc = check_step_rows(who, "du", a->T, a->B, a->H, a->sdu_t, a->sdu_b, true))) return rc;
  if ((rc = check_step_rows(who, "ddelta", a->T, a->B, a->H, a->sdd_t, a->sdd_b, true))) return rc;
  return a->z ? check_step_rows(who, "dz", a->T, a->B, a->H, a->sdz_t, a->sdz_b, true) : GS_OK;
}

template <typename Args>
SsmParams params_of(const Args* a, const Plan& plan, const Bytes& bytes) {
  SsmParams p{};
  p.u = a->u;
  p.delta = a->delta;
  p.z = a->z;
  p.bm = a->bm;
  p.cm = a->cm;
  p.A = a->A;
  p.D = a->D;
  p.bias = a->delta_bias;
  p.h0 = a->h0;
  p.reset = a->reset;
  p.su_t = a->su_t;
  p.su_b = a->su_b;
  p.sdl_t = a->sdl_t;
  p.sdl_b = a->sdl_b;
  p.sz_t = a->sz_t;
  p.sz_b = a->sz_b;
  p.sb_t = a->sb_t;
  p.sb_b = a->sb_b;
  p.sc_t = a->sc_t;
  p.sc_b = a->sc_b;
  p.sr_t = a->sr_t;
  p.sr_b = a->sr_b;
  p.T = (int)a->T;
  p.B = (int)a->B;
  p.H = (int)a->H;
  p.N = (int)a->N;
  p.blocks = plan.blocks;
  p.chunks = plan.chunks;
  p.length = plan.length;
  p.each = plan.each;
  char* s = static_cast<char*>(a->scratch);
  p.ends = reinterpret_cast<float*>(s + bytes.ends);
  p.span = reinterpret_cast<float*>(s + bytes.span);
  p.part_bc = reinterpret_cast<float*>(s + bytes.bc);
  p.part_a = reinterpret_cast<float*>(s + bytes.a);
  return p;
}

int join_ends(const SsmParams& p, bool back, hipStream_t stream) {
  const int64_t n = (int64_t)p.B * p.N * p.H;
  hipLaunchKernelGGL(back ? ssm_join_kernel<true> : ssm_join_kernel<false>, dim3((unsigned)((n + 63) / 64)), dim3(64), 0,
                     stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}

// What a training forward keeps: states, and behind them the outputs before their gate.
template <typename Args>
int64_t saved_states(const Args* a) {
  return (a->T + kTile - 1) / kTile * a->B * a->N * a->H;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int64_t gs_ssm_scratch_bytes(const gs_ssm_args* a) {
  clear_error();
  const int rc = check_fwd(a, "gs_ssm_scratch_bytes");
  return rc ? rc : bytes_of(make_plan(a->T, a->B, a->H, false), a->T, a->B, a->H, a->N, false).total;
}

extern "C" int64_t gs_ssm_saved_bytes(const gs_ssm_args* a) {
  clear_error();
  const int rc = check_fwd(a, "gs_ssm_saved_bytes");
  return rc ? rc : (saved_states(a) + (a->z ? a->T * a->B * a->H : 0)) * 4;
}

extern "C" int gs_ssm_fwd(const gs_ssm_args* a, hipStream_t stream) {
  const char* who = "gs_ssm_fwd";
  clear_error();
  int rc = check_fwd(a, who);
  if (rc) return rc;
  if (!a->u || !a->delta || !a->bm || !a->cm || !a->A || !a->y)
    return set_error(GS_ERR_INVALID, "%s: u, delta, A, bm, cm and y must be non-NULL device pointers", who);
  const Plan plan = make_plan(a->T, a->B, a->H, false);
  const Bytes bytes = bytes_of(plan, a->T, a->B, a->H, a->N, false);
  if ((rc = check_plain_scratch(who, a->scratch, a->scratch_bytes, bytes.total))) return rc;
  SsmParams p = params_of(a, plan, bytes);
  p.y = a->y;
  p.h_last = a->h_last;
  p.saved = a->saved;
  p.ungated = a->saved && a->z ? a->saved + saved_states(a) : nullptr;
  p.sy_t = a->sy_t;
  p.sy_b = a->sy_b;
  const int64_t groups = (int64_t)plan.blocks * a->B * std::max(1, plan.chunks - 1);
  if (plan.chunks > 1) {
    if ((rc = launch(kFwdFirst, plan.wide, a->dtype, p, groups, stream))) return rc;
    if (plan.chunks > 2 && (rc = join_ends(p, false, stream))) return rc;
  }
  return launch(kFwd, plan.wide, a->dtype, p, groups, stream);
}

extern "C" int64_t gs_ssm_bwd_scratch_bytes(const gs_ssm_bwd_args* a) {
  clear_error();
  const int rc = check_bwd(a, "gs_ssm_bwd_scratch_bytes");
  return rc ? rc : bytes_of(make_plan(a->T, a->B, a->H, true), a->T, a->B, a->H, a->N, true).total;
}

extern "C" int gs_ssm_bwd(const gs_ssm_bwd_args* a, hipStream_t stream) {
  const char* who = "gs_ssm_bwd";
  clear_error();
  int rc = check_bwd(a, who);
  if (rc) return rc;
  if (!a->u || !a->delta || !a->bm || !a->cm || !a->A || !a->saved || !a->dy || !a->du || !a->ddelta || (a->z && !a->dz))
    return set_error(GS_ERR_INVALID, "%s: u, delta, A, bm, cm, saved, dy, du and ddelta (and dz where z is given) must be "
                     "non-NULL device pointers", who);
  const Plan plan = make_plan(a->T, a->B, a->H, true);
  const Bytes bytes = bytes_of(plan, a->T, a->B, a->H, a->N, true);
  if ((rc = check_plain_scratch(who, a->scratch, a->scratch_bytes, bytes.total))) return rc;
  SsmParams p = params_of(a, plan, bytes);
  p.saved = const_cast<float*>(a->saved);
  p.ungated = a->z ? p.saved + saved_states(a) : nullptr;
  p.dy = a->dy;
  p.dh_last = a->dh_last;
  p.du = a->du;
  p.ddelta = a->ddelta;
  p.dz = a->dz;
  p.dh0 = a->dh0;
  p.sdy_t = a->sdy_t;
  p.sdy_b = a->sdy_b;
  p.sdu_t = a->sdu_t;
  p.sdu_b = a->sdu_b;
  p.sdd_t = a->sdd_t;
  p.sdd_b = a->sdd_b;
  p.sdz_t = a->sdz_t;
  p.sdz_b = a->sdz_b;
  const int64_t groups = (int64_t)plan.blocks * a->B, rows = a->T * a->B;
  if (plan.chunks > 1) {
    const int64_t part = plan.length / plan.each, parts = (a->T + part - 1) / part;
    if ((rc = launch(kBwdEnds, plan.wide, a->dtype, p, groups * (parts - plan.each), stream))) return rc;
    if ((rc = join_ends(p, true, stream))) return rc;
  }
  if ((rc = launch(kBwd, plan.wide, a->dtype, p, groups * plan.chunks, stream))) return rc;
  const int bc_groups = (int)std::min<int64_t>((rows * 2 * a->N + 255) / 256, 1 << 20);
  const SumParams sums{p.part_bc, p.part_a, a->dbm, a->dcm, a->dA, a->dD, a->ddelta_bias, rows, (int)a->H, (int)a->N, plan.blocks,
                       (int)(plan.chunks * a->B), bc_groups};
  hipLaunchKernelGGL(a->dtype == GS_DTYPE_F32 ? ssm_sum_kernel<float> : ssm_sum_kernel<__bf16>,
                     dim3((unsigned)(bc_groups + plan.blocks * (a->N + 2))), dim3(256), 0, stream, sums);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}

extern "C" int gs_ssm_step(const gs_ssm_step_args* a, hipStream_t stream) {
  const char* who = "gs_ssm_step";
  clear_error();
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  const int rc = check_sizes(who, 1, a->B, a->H, a->N, a->dtype);
  if (rc) return rc;
  if (!a->u || !a->delta || !a->bm || !a->cm || !a->A || !a->state || !a->y)
    return set_error(GS_ERR_INVALID, "%s: u, delta, A, bm, cm, state and y must be non-NULL device pointers", who);
  if (a->S < 1 || a->S > (1ll << 30) || (a->slots == nullptr && a->S < a->B))
    return set_error(GS_ERR_INVALID, "%s: a cache of S=%lld states does not hold B=%lld rows", who, (long long)a->S,
                     (long long)a->B);
  if (a->su < 0 || a->sdl < 0 || a->sz < 0 || a->sb < 0 || a->sc < 0 || (a->S > 1 && a->ss < a->H * a->N) ||
      (a->B > 1 && a->sy < a->H))
    return set_error(GS_ERR_INVALID, "%s: strides do not describe rows of H=%lld and states of [H, N]", who, (long long)a->H);
  if (a->B > 65535) return set_error(GS_ERR_INVALID, "%s: B=%lld exceeds 65535", who, (long long)a->B);
  SsmStepParams p{a->u, a->delta, a->z, a->bm, a->cm, a->A, a->D, a->delta_bias, a->state, a->slots, a->y,
                  a->su, a->sdl, a->sz, a->sb, a->sc, a->ss, a->sy, (int)a->B, (int)a->H, (int)a->N, (int)a->S};
  const bool vec = a->N % 4 == 0 && a->ss % 4 == 0 &&
                   ((reinterpret_cast<uintptr_t>(a->A) | reinterpret_cast<uintptr_t>(a->state)) & 15u) == 0;
  void (*fn)(SsmStepParams) = a->dtype == GS_DTYPE_F32 ? (vec ? ssm_step_kernel<float, true> : ssm_step_kernel<float, false>)
                                                       : (vec ? ssm_step_kernel<__bf16, true> : ssm_step_kernel<__bf16, false>);
  hipLaunchKernelGGL(fn, dim3((unsigned)((a->H + 63) / 64), (unsigned)a->B), dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}
