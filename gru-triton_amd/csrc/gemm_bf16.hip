// bf16 products on v_mfma_f32_16x16x32_bf16 (gfx950) for the linear operator: x w^T
// (NT), dpre w (NN) and dpre^T x (TN), with the bias, activation and residual of the
// forward in the epilogue.
//
// A workgroup computes a T x T tile of C, T = 256 with 8 waves (each 128 x 64 of it) or
// 128 or 64 with 4 (each a quarter), K in slices of 32. The MFMA takes B's tile as its
// first operand, so that a lane holds four consecutive columns of one row of C (D VGPR v
// of lane l: C[l % 16][4 (l / 16) + v]) and stores them at once. While a slice's products
// run, the next slice's operands are read from LDS into a second set of registers, so that
// after the barrier that ends a slice the matrix pipe goes on at once. 8192 x 8192 x 8192
// takes 840 us forward and 760 for either gradient (1.3 and 1.45 PFLOP/s), bound by the
// matrix pipe.
//
// LDS layouts (16-byte granules, no padding):
//   operand contiguous along k: row r is 4 granules of 8 k; granule c sits in slot
//     c ^ swz(r). A lane reads k = 8 (l / 16) of row l % 16 in 16 bytes; the 16 lanes of
//     a pass (rows r < 8 of one k-group and r >= 8 of another) then cover all 64 banks.
//   operand contiguous along its rows: k-row k is R / 8 granules of 8 rows; granule g
//     sits in slot g ^ swz(k). ds_read_b64_tr_b16 gives lane l of each 16 four
//     consecutive k of row l % 16 (lane l supplies the address of k = l / 4, rows
//     4 (l % 4) .. + 3); the 8 k-rows that a pass of 32 lanes touches (k % 4 and bit 3
//     of k) sit in different 32-byte bank groups.
// Operands whose rows are 16-byte aligned come straight from memory to LDS
// (buffer_load ... lds, 16 bytes a lane; the swizzle is in the address each lane asks
// for, a lane past an edge asks for an offset out of range and gets zeros), four slices
// deep. Others go through registers, in 16-byte loads at any address, element by element
// where a granule crosses the end of a row.
#include "gs_gemm_bf16.h"

namespace gs {
namespace {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void LdsVoid;
typedef __attribute__((address_space(3))) s4v LdsS4;

constexpr int BK = 32;

// One operand's tile of a slice: R rows x BK k in LDS.
template <int R, bool KC, int THREADS>
struct Tile {
  static constexpr int kBytes = R * BK * 2;
  static constexpr int kLoads = kBytes / 16 / THREADS;  // granules of a thread
  static constexpr int kReads = KC ? 1 : 2;              // LDS reads of a fragment
  static_assert(kLoads >= 1, "a granule for every thread");

  static __device__ __forceinline__ int swz(int x) {  // of a row (KC) or a k
    if constexpr (KC) return ((x >> 2) & 3) ^ ((x >> 3) & 1);
    return R >= 128 ? 2 * ((x & 3) | ((x >> 1) & 4)) : 2 * (((x >> 1) & 1) | ((x >> 2) & 2));
  }
  // row (the first of 8, if not KC) and k (the first of 8, if KC) of the granule at byte `at` of the tile
  static __device__ __forceinline__ void granule(int at, int* row, int* k) {
    if constexpr (KC) {
      *row = at >> 6;
      *k = (((at >> 4) & 3) ^ swz(*row)) * 8;
    } else {
      *k = at / (2 * R);
      *row = (((at % (2 * R)) >> 4) ^ swz(*k)) * 8;
    }
  }
  // rows row0 .. row0 + 15 (row0 a multiple of 16) of the slice, as an MFMA takes them
  static __device__ __forceinline__ bf8 fragment(const char* lds, int row0, int lane) {
    const int r = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      return *reinterpret_cast<const bf8*>(lds + (row0 + r) * 64 + ((g ^ swz(r)) << 4));
    } else {
      const int k = 8 * g + (r >> 2);  // and k + 4: the same swz
      const int at = k * 2 * R + ((((row0 >> 3) + ((r & 3) >> 1)) ^ swz(k)) << 4) + ((r & 1) << 3);
      union {
        s4v h[2];
        bf8 v;
      } u;
#pragma unroll
      for (int h = 0; h < 2; ++h) u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4*)(lds + at + h * 8 * R));
      return u.v;
    }
  }
};

// Straight to LDS. Rows and k that do not exist, and slices from n on, load zeros.
template <int R, bool KC, int THREADS>
struct Direct : Tile<R, KC, THREADS> {
  typedef Tile<R, KC, THREADS> T;
  const __bf16* base;
  int64_t step;
  uint32_t off[T::kLoads], tail[T::kLoads];
  __device__ __forceinline__ void init(const __bf16* p, int64_t ld, int row0, int lim, int kbeg, int klast, int kend) {
    base = KC ? p + (int64_t)row0 * ld + kbeg : p + (int64_t)kbeg * ld + row0;
    step = KC ? BK : BK * ld;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < T::kLoads; ++e) {
      int row, k;
      T::granule((wave * T::kLoads + e) * 1024 + lane * 16, &row, &k);
      off[e] = row0 + row < lim ? (uint32_t)(2 * (KC ? row * ld + k : k * ld + row)) : kOffNone;
      tail[e] = klast + k < kend ? 0u : kOffNone;
    }
  }
  __device__ __forceinline__ void load(int s, int n, char* lds) const {
    const uint32_t last = s == n - 1 ? ~0u : 0u, past = s >= n ? kOffNone : 0u;
    const auto r = bounded_rsrc(base + s * step, 0x7fffffffu);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int e = 0; e < T::kLoads; ++e)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsVoid*)(lds + (wave * T::kLoads + e) * 1024), 16,
                                               (int)(off[e] | (tail[e] & last) | past), 0, 0, 0);
  }
};

// Through registers.
template <int R, bool KC, int THREADS>
struct Staged : Tile<R, KC, THREADS> {
  typedef Tile<R, KC, THREADS> T;
  const __bf16* p;
  int64_t ld;
  int row0, lim, kbeg, kend;
  __device__ __forceinline__ void init(const __bf16* p_, int64_t ld_, int row0_, int lim_, int kbeg_, int, int kend_) {
    p = p_;
    ld = ld_;
    row0 = row0_;
    lim = lim_;
    kbeg = kbeg_;
    kend = kend_;
  }
  __device__ __forceinline__ bool inside(int s) const {  // uniform
    return row0 + R <= lim && kbeg + s * BK + BK <= kend;
  }
  // elements of granule e of slice s that exist, along the contiguous side
  __device__ __forceinline__ int have(int s, int e, int* row, int* k) const {
    T::granule((threadIdx.x + e * THREADS) * 16, row, k);
    const int r = row0 + *row, kk = kbeg + s * BK + *k;
    return KC ? (r < lim ? kend - kk : 0) : (kk < kend ? lim - r : 0);
  }
  __device__ __forceinline__ void load(int s, Granule (&x)[T::kLoads]) const {
    const int k0 = kbeg + s * BK;
    const __bf16* base = KC ? p + (int64_t)row0 * ld + k0 : p + (int64_t)k0 * ld + row0;
    const bool in = inside(s);
#pragma unroll
    for (int e = 0; e < T::kLoads; ++e) {
      int row, k;
      const int h = have(s, e, &row, &k);
      const __bf16* q = base + (KC ? row * ld + k : k * ld + row);
      if (in)
        x[e] = *reinterpret_cast<const GranuleAt*>(q);
      else
        x[e] = granule_load(q, h, KC ? k0 + k : row0 + row);
    }
  }
  __device__ __forceinline__ void stage(int s, char* lds, Granule (&x)[T::kLoads]) const {
    const bool in = inside(s);
#pragma unroll
    for (int e = 0; e < T::kLoads; ++e) {
      int row, k;
      if (!in) x[e] = granule_settle(x[e], have(s, e, &row, &k));
      *reinterpret_cast<Granule*>(lds + (threadIdx.x + e * THREADS) * 16) = x[e];
    }
  }
};

// Eight elements of a row from column j on, as far as they exist, at any alignment.
__device__ __forceinline__ void load_row8(const void* row, int j, int N, float (&x)[8]) {
  granule_floats(granule_settle(granule_load(static_cast<const __bf16*>(row) + j, N - j, j), N - j), x);
}
__device__ __forceinline__ void store_row8(void* row, int j, int N, const float (&x)[8]) {
  __bf16* p = static_cast<__bf16*>(row) + j;
  if (j + 8 <= N) {
    GranuleAt w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = __builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{x[2 * i], x[2 * i + 1]}), bf2v));
    *reinterpret_cast<GranuleAt*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (j + i < N) p[i] = (__bf16)x[i];
  }
}

// A row's eight elements of pre from column j on, as the backward takes them.
__device__ __forceinline__ void keep_row8(void* row, int j, int N, const float (&x)[8]) {
  GranuleAt w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = kept_pair(x[2 * i], x[2 * i + 1]);
  unsigned short* p = static_cast<unsigned short*>(row) + j;
  if (j + 8 <= N) {
    *reinterpret_cast<GranuleAt*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (j + i < N) p[i] = (unsigned short)(w[i >> 1] >> (16 * (i & 1)));
  }
}

// What follows the sums of columns j .. j + 7 of row i (< M; columns from N on do not exist).
__device__ __forceinline__ void finish8(const LinearEpilogue& e, __bf16* y, int64_t ldy, int i, int j, int N,
                                        const float (&bias)[8], float (&x)[8]) {
#pragma unroll
  for (int v = 0; v < 8; ++v) x[v] += bias[v];
  if (e.pre != nullptr) keep_row8(static_cast<unsigned short*>(e.pre) + (int64_t)i * N, j, N, x);
  if (e.act != GS_ACT_NONE) act_values(x, e.act);
  if (e.residual != nullptr) {
    float r[8];
    load_row8(static_cast<const __bf16*>(e.residual) + i * e.ldr, j, N, r);
#pragma unroll
    for (int v = 0; v < 8; ++v) x[v] += r[v];
  }
  store_row8(y + i * ldy, j, N, x);
}

// The order of a slice's NM MFMAs and, between them, NR LDS reads, NW LDS writes and NV
// loads: the reads first, one per MFMA or two, then the others.
template <int NM, int NR, int NW, int NV>
__device__ __forceinline__ void interleave() {
  constexpr int kPer = NR * 4 <= NM * 3 ? 1 : 2, kFirst = (NR + kPer - 1) / kPer;
  constexpr int kRest = NM - kFirst > 0 ? NM - kFirst : 1, kPut = (NW + NV + kRest - 1) / kRest;
  static_for<0, NM>([&](auto I) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
    if constexpr (I < kFirst) {
      __builtin_amdgcn_sched_group_barrier(0x100, kPer, 0);  // LDS read
    } else {
      constexpr int at = (I - kFirst) * kPut;
      if constexpr (at < NW) __builtin_amdgcn_sched_group_barrier(0x200, kPut, 0);
      if constexpr (at >= NW && at < NW + NV) __builtin_amdgcn_sched_group_barrier(0x020, kPut, 0);
    }
  });
}

// What a launch stores: finished outputs, a split's sums, or either as it is asked. TN
// products take the last: with the first two apart, the instance of 256 x 256 tiles that
// stores sums spilled inside its loop (128 slices in 166 us instead of 100); the others
// store finished outputs faster alone (M = 32768, N = 2048, K = 1024: 136 us, not 147).
enum { kOutputs = 0, kSums = 1, kEither = 2 };

// LDS of a product's tiles: four slices of each operand (two where they come through
// registers), as arrays of their own, so that the compiler knows which loads to LDS a read
// has to wait for.
#define GS_TILE_LDS(BT)                                                                            \
  __shared__ __attribute__((aligned(1024))) char A0[(BT)*BK * 2], A1[(BT)*BK * 2], A2[(BT)*BK * 2], \
      A3[(BT)*BK * 2], B0[(BT)*BK * 2], B1[(BT)*BK * 2], B2[(BT)*BK * 2], B3[(BT)*BK * 2]
#define GS_TILE_ARRAYS A0, A1, A2, A3, B0, B1, B2, B3

// Workgroup `group` of a product. Its waves are 2 along the rows by WJ along the columns.
template <int BT, int WJ, int LAYOUT, bool DIRECT, int PART>
__device__ __forceinline__ void gemm_bf16_group(const GemmBf16Args& g, int group, char* A0, char* A1, char* A2, char* A3,
                                                char* B0, char* B1, char* B2, char* B3) {
  constexpr int THREADS = 128 * WJ, TI = BT / 32, TJ = BT / WJ / 16;  // a wave's fragments
  constexpr bool A_KC = LAYOUT != kGemmTN, B_KC = LAYOUT == kGemmNT;
  typedef typename std::conditional<DIRECT, Direct<BT, A_KC, THREADS>, Staged<BT, A_KC, THREADS>>::type LA;
  typedef typename std::conditional<DIRECT, Direct<BT, B_KC, THREADS>, Staged<BT, B_KC, THREADS>>::type LB;
  constexpr int kLoads = LA::kLoads + LB::kLoads;
  // Each XCD (workgroup mod 8) takes one split, or as few as there are, and of its tiles a
  // run, in patches of 1024 rows: its L2 then holds what its workgroups share. (With the
  // tiles of every split spread over all XCDs, dw of M = 32768, N = 2048, K = 1024 read
  // 670 MB instead of 200.)
  const int mt = (g.M + BT - 1) / BT, nt = (g.N + BT - 1) / BT, total = mt * nt;
  const int xcd = group & 7, spread = g.ksplit < 8 ? 8 / g.ksplit : 1;  // XCDs of a split
  const int per = (total + spread - 1) / spread, slot = group >> 3;
  const int split = g.ksplit < 8 ? xcd % g.ksplit : xcd + 8 * (slot / per);
  const int tile = g.ksplit < 8 ? xcd / g.ksplit * per + slot : slot % per;
  if ((g.ksplit < 8 && slot >= per) || split >= g.ksplit || tile >= total) return;  // uniform
  constexpr int kPatch = 1024 / BT;
  const int patch = tile / (kPatch * nt), in_patch = tile - patch * kPatch * nt;
  const int pm = min(kPatch, mt - patch * kPatch);
  const int i0 = (patch * kPatch + in_patch % pm) * BT, j0 = in_patch / pm * BT;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / WJ * (BT / 2), wj = wave % WJ * (BT / WJ);
  const int kper = ((g.K + g.ksplit - 1) / g.ksplit + BK - 1) / BK * BK;
  const int kbeg = split * kper, kend = min(g.K, kbeg + kper);
  const int n = kend > kbeg ? (kend - kbeg + BK - 1) / BK : 0;

  LA la;
  LB lb;
  la.init(g.a, g.lda, i0, g.M, kbeg, kbeg + (n - 1) * BK, kend);
  lb.init(g.b, g.ldb, j0, g.N, kbeg, kbeg + (n - 1) * BK, kend);

  f4v acc[TI][TJ];
#pragma unroll
  for (int a = 0; a < TI; ++a)
#pragma unroll
    for (int b = 0; b < TJ; ++b) acc[a][b] = f4v{0.f, 0.f, 0.f, 0.f};
  struct Operands {
    bf8 a[TI], b[TJ];
  };
  Operands f0, f1;
  auto read = [&](const char* A, const char* B, Operands& f) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < TJ; ++b) f.b[b] = LB::fragment(B, wj + 16 * b, lane);
#pragma unroll
    for (int a = 0; a < TI; ++a) f.a[a] = LA::fragment(A, wi + 16 * a, lane);
  };
  auto products = [&](const Operands& f) __attribute__((always_inline)) {
#pragma unroll
    for (int a = 0; a < TI; ++a)
#pragma unroll
      for (int b = 0; b < TJ; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.b[b], f.a[a], acc[a][b], 0, 0, 0);
  };
  constexpr int kReads = TI * LA::kReads + TJ * LB::kReads;
  if constexpr (DIRECT) {
    auto load = [&](int s, char* A, char* B) __attribute__((always_inline)) {
      la.load(s, n, A);
      lb.load(s, n, B);
    };
    // All but the last `kYoung` slices loaded have arrived for every wave, and this wave's
    // LDS reads are done: two slices stay in flight across a barrier.
    auto arrive = [&](auto young) __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(decltype(young)::value * kLoads) : "memory");
    };
    constexpr std::integral_constant<int, 2> I2{};
    constexpr std::integral_constant<int, 3> I3{};
    load(0, A0, B0);
    load(1, A1, B1);
    load(2, A2, B2);
    load(3, A3, B3);
    arrive(I3);
    read(A0, B0, f0);
    arrive(I2);
    // Slice s: its operands are in registers; slice s + 1 has arrived and is read; slice
    // s + 4 goes where s was, which every wave read before the last barrier.
    auto slice = [&](int s, const Operands& f, Operands& next, const char* A, const char* B, char* Af,
                     char* Bf) __attribute__((always_inline)) {
      read(A, B, next);
      load(s + 4, Af, Bf);
      products(f);
      interleave<TI * TJ, kReads, 0, kLoads>();
      arrive(I2);
    };
    for (int s = 0; s < n; s += 4) {  // slices from n on are zeros
      slice(s, f0, f1, A1, B1, A0, B0);
      slice(s + 1, f1, f0, A2, B2, A1, B1);
      slice(s + 2, f0, f1, A3, B3, A2, B2);
      slice(s + 3, f1, f0, A0, B0, A3, B3);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load to LDS outlives the workgroup
  } else {
    Granule xa[2][LA::kLoads], xb[2][LB::kLoads];
    auto load = [&](int s, auto I) __attribute__((always_inline)) {
      la.load(s, xa[I]);
      lb.load(s, xb[I]);
    };
    auto put = [&](int s, auto I, char* A, char* B) __attribute__((always_inline)) {  // slice s to LDS, its registers take s + 2
      la.stage(s, A, xa[I]);
      lb.stage(s, B, xb[I]);
      load(s + 2, I);
    };
    constexpr std::integral_constant<int, 0> I0{};
    constexpr std::integral_constant<int, 1> I1{};
    load(0, I0);
    load(1, I1);
    put(0, I0, A0, B0);
    put(1, I1, A1, B1);
    lds_barrier();
    read(A0, B0, f0);
    lds_barrier();
    auto slice = [&](int s, auto I, const Operands& f, Operands& next, const char* A, const char* B, char* Af,
                     char* Bf) __attribute__((always_inline)) {
      read(A, B, next);
      put(s + 2, I, Af, Bf);
      products(f);
      interleave<TI * TJ, kReads, kLoads, kLoads>();
      lds_barrier();
    };
    for (int s = 0; s < n; s += 2) {
      slice(s, I0, f0, f1, A1, B1, A0, B0);
      slice(s + 1, I1, f1, f0, A0, B0, A1, B1);
    }
  }

  // Each wave passes its part of C through LDS, 16 rows at a time, so that a lane gets
  // eight consecutive columns of a row and a row's bytes are stored together: stored as
  // the MFMA leaves them (8 bytes a lane, 32 of a row at once), the epilogue of M = 32768,
  // N = 2048 took 93 us.
  constexpr int kCols = 16 * TJ, kStride = kCols + 4, kLanes = kCols / 8;  // kLanes lanes hold a row
  static_assert(16 * kStride * 4 <= LA::kBytes / (THREADS / 256), "a wave's share of a buffer");
  lds_barrier();  // every wave has read its last operands
  char* room;
  if constexpr (DIRECT)
    room = (wave & 3) == 0 ? A0 : (wave & 3) == 1 ? A1 : (wave & 3) == 2 ? B0 : B1;
  else
    room = wave == 0 ? A0 : wave == 1 ? A1 : wave == 2 ? B0 : B1;
  float* mine = reinterpret_cast<float*>(room + (wave >> 2) * (LA::kBytes / (THREADS / 256)));
  const int r16 = lane & 15, q4 = (lane >> 4) * 4;
  const int j = j0 + wj + 8 * (lane % kLanes);
  float bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (PART != kSums && g.epi.bias != nullptr && j < g.N) load_row8(g.epi.bias, j, g.N, bias);
#pragma unroll
  for (int a = 0; a < TI; ++a) {
#pragma unroll
    for (int b = 0; b < TJ; ++b) *reinterpret_cast<f4v*>(mine + r16 * kStride + 16 * b + q4) = acc[a][b];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (PART == kSums || (PART == kEither && g.ksplit > 1)) {  // four columns a lane: a store covers whole lines
      typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
      constexpr int kQuads = kCols / 4;
      const int jq = j0 + wj + 4 * (lane % kQuads);
#pragma unroll
      for (int rr = 0; rr < 16; rr += 64 / kQuads) {
        const int row = rr + lane / kQuads, i = i0 + wi + 16 * a + row;
        const f4v w = *reinterpret_cast<const f4v*>(mine + row * kStride + 4 * (lane % kQuads));
        if (i >= g.M || jq >= g.N) continue;
        float* c = g.part + ((int64_t)split * g.M + i) * g.N + jq;
        if (jq + 4 <= g.N) {
          *reinterpret_cast<f4u*>(c) = w;
        } else {
#pragma unroll
          for (int v = 0; v < 3; ++v)
            if (jq + v < g.N) c[v] = w[v];
        }
      }
    } else {
#pragma unroll
      for (int rr = 0; rr < 16; rr += 64 / kLanes) {
        const int row = rr + lane / kLanes, i = i0 + wi + 16 * a + row;
        float x[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f4v w = *reinterpret_cast<const f4v*>(mine + row * kStride + 8 * (lane % kLanes) + 4 * h);
#pragma unroll
          for (int v = 0; v < 4; ++v) x[4 * h + v] = w[v];
        }
        if (i >= g.M || j >= g.N) continue;
        finish8(g.epi, g.y, g.ldy, i, j, g.N, bias, x);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <int BT, int WJ, int LAYOUT, bool DIRECT, int PART>
__global__ __launch_bounds__(128 * WJ, 2) void gemm_bf16_kernel(GemmBf16Args g) {
  if constexpr (DIRECT) {
    GS_TILE_LDS(BT);
    gemm_bf16_group<BT, WJ, LAYOUT, DIRECT, PART>(g, blockIdx.x, GS_TILE_ARRAYS);
  } else {
    __shared__ __attribute__((aligned(1024))) char A0[BT * BK * 2], A1[BT * BK * 2], B0[BT * BK * 2], B1[BT * BK * 2];
    gemm_bf16_group<BT, WJ, LAYOUT, DIRECT, PART>(g, blockIdx.x, A0, A1, nullptr, nullptr, B0, B1, nullptr, nullptr);
  }
}

// The products of a small backward in one launch, side by side on the device: dx (NN),
// dw (TN) and the column sums' end (sum_columns) have no part in each other.
template <bool DIRECT>
__global__ __launch_bounds__(256, 2) void gemm_bf16_pair_kernel(GemmBf16Args x, GemmBf16Args w, ColumnSums c, int nx, int nw) {
  const int group = blockIdx.x;
  if constexpr (DIRECT) {
    GS_TILE_LDS(64);
    if (group < nw)
      gemm_bf16_group<64, 2, kGemmTN, DIRECT, kEither>(w, group, GS_TILE_ARRAYS);
    else if (group < nw + nx)
      gemm_bf16_group<64, 2, kGemmNN, DIRECT, kOutputs>(x, group - nw, GS_TILE_ARRAYS);
    else
      sum_columns<__bf16>(c, group - nw - nx, reinterpret_cast<float(*)[17]>(A0));
  } else {
    __shared__ __attribute__((aligned(1024))) char A0[64 * BK * 2], A1[64 * BK * 2], B0[64 * BK * 2], B1[64 * BK * 2];
    if (group < nw)
      gemm_bf16_group<64, 2, kGemmTN, DIRECT, kEither>(w, group, A0, A1, nullptr, nullptr, B0, B1, nullptr, nullptr);
    else if (group < nw + nx)
      gemm_bf16_group<64, 2, kGemmNN, DIRECT, kOutputs>(x, group - nw, A0, A1, nullptr, nullptr, B0, B1, nullptr, nullptr);
    else
      sum_columns<__bf16>(c, group - nw - nx, reinterpret_cast<float(*)[17]>(A0));
  }
}

// y from the splits' sums, added in order: eight columns a thread, the loads of up to
// eight splits in flight.
__global__ __launch_bounds__(256) void gemm_bf16_finish_kernel(GemmBf16Args g) {
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  const int octets = (g.N + 7) / 8;
  const int64_t all = (int64_t)g.M * octets, stride = (int64_t)g.M * g.N;
  for (int64_t q = blockIdx.x * (int64_t)256 + threadIdx.x; q < all; q += (int64_t)gridDim.x * 256) {
    const int i = (int)(q / octets), j = (int)(q - (int64_t)i * octets) * 8;
    float x[8], bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < 8; ++v) x[v] = 0.0f;
    const float* c = g.part + (int64_t)i * g.N + j;
    for (int s = 0; s < g.ksplit; s += 8) {
      f4u w[8][2];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const float* d = c + (s + u) * stride;
        w[u][0] = w[u][1] = f4u{0.f, 0.f, 0.f, 0.f};
        if (s + u >= g.ksplit) continue;
        if (j + 8 <= g.N) {
          w[u][0] = *reinterpret_cast<const f4u*>(d);
          w[u][1] = *reinterpret_cast<const f4u*>(d + 4);
        } else {
#pragma unroll
          for (int v = 0; v < 8; ++v)
            if (j + v < g.N) w[u][v >> 2][v & 3] = d[v];
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int v = 0; v < 8; ++v) x[v] += w[u][v >> 2][v & 3];
    }
    if (g.epi.bias != nullptr) load_row8(g.epi.bias, j, g.N, bias);
    finish8(g.epi, g.y, g.ldy, i, j, g.N, bias, x);
  }
}

// ---- few rows ------------------------------------------------------------------------
// x w^T for at most 16 MT rows of x, as in serving: what there is to do is to read w once.
// A workgroup takes 16 columns; its 8 waves take K in turns of 32 and hold the operands
// of kAhead turns straight from memory, without LDS; their sums are joined through LDS in
// order. M = 8, N = 2048, K = 1024: 4.1 us on the GPU, 1.0 TB/s of w, where an empty launch
// takes 2.3; in 64 x 64 tiles (32 workgroups, 32 slices one after the other) 6.4.
constexpr int kRowWaves = 8;
template <int MT>
__global__ __launch_bounds__(64 * kRowWaves) void gemm_bf16_rows_kernel(GemmBf16Args g) {
  constexpr int kAhead = 4;
  __shared__ __attribute__((aligned(16))) float red[kRowWaves][MT][64 * 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4, n0 = blockIdx.x * 16;
  const bool whole = g.K % 32 == 0;  // uniform: no granule crosses the end of a row
  const __bf16* w = g.b + (int64_t)min(n0 + r, g.N - 1) * g.ldb;  // past the edge: a row that exists, not stored
  const __bf16* x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) x[t] = g.a + (int64_t)min(16 * t + r, g.M - 1) * g.lda;
  f4v acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f4v{0.f, 0.f, 0.f, 0.f};
  auto run = [&](auto WHOLE) __attribute__((always_inline)) {
    constexpr bool in = decltype(WHOLE)::value;
    for (int k0 = wave * 32; k0 < g.K; k0 += kRowWaves * 32 * kAhead) {
      Granule fw[kAhead], fx[kAhead][MT];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = k0 + u * kRowWaves * 32 + 8 * q;
        if (in) {
          const int kk = min(k, g.K - 8);  // past the end: not used
          fw[u] = *reinterpret_cast<const GranuleAt*>(w + kk);
#pragma unroll
          for (int t = 0; t < MT; ++t) fx[u][t] = *reinterpret_cast<const GranuleAt*>(x[t] + kk);
        } else {
          fw[u] = granule_load(w + k, g.K - k, k);
#pragma unroll
          for (int t = 0; t < MT; ++t) fx[u][t] = granule_load(x[t] + k, g.K - k, k);
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int k = k0 + u * kRowWaves * 32;
        if (k >= g.K) break;  // uniform
        if (!in) fw[u] = granule_settle(fw[u], g.K - k - 8 * q);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if (!in) fx[u][t] = granule_settle(fx[u][t], g.K - k - 8 * q);
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, fw[u]), __builtin_bit_cast(bf8, fx[u][t]),
                                                           acc[t], 0, 0, 0);
        }
      }
    }
  };
  if (whole)
    run(std::true_type{});
  else
    run(std::false_type{});
#pragma unroll
  for (int t = 0; t < MT; ++t) *reinterpret_cast<f4v*>(&red[wave][t][lane * 4]) = acc[t];
  __syncthreads();
  // eight columns a thread: row i, columns 8 h .. 8 h + 7 of the workgroup's 16
  const int i = threadIdx.x >> 1, h = threadIdx.x & 1, j = n0 + 8 * h;
  if (i >= 16 * MT || i >= g.M || j >= g.N) return;
  float y[8], bias[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int v = 0; v < 8; ++v) y[v] = 0.0f;
#pragma unroll
  for (int wv = 0; wv < kRowWaves; ++wv)
#pragma unroll
    for (int v = 0; v < 8; ++v) y[v] += red[wv][i >> 4][((i & 15) + 16 * (2 * h + (v >> 2))) * 4 + (v & 3)];
  if (g.epi.bias != nullptr) load_row8(g.epi.bias, j, g.N, bias);
  finish8(g.epi, g.y, g.ldy, i, j, g.N, bias, y);
}

// ---- host ---------------------------------------------------------------------------

int64_t tiles_of(int M, int N, int T) { return (int64_t)((M + T - 1) / T) * ((N + T - 1) / T); }

constexpr int kTileSizes[3] = {256, 128, 64};

// Microseconds of a product with tile T and `split` splits of K, from runs on the chip:
// a launch takes 3; a CU does a tile's slice in `slice` and its first loads and last
// stores in `ends`, tile after tile; splits write their sums and a second launch reads
// them. Rows M, N, K of x w^T, dpre w and dpre^T x; measured (predicted) in us:
//                         T = 256          T = 128       T = 64
//   32768, 2048, 1024 fwd 141 (128)        162 (167)     241 (243)
//   32768, 2048, 1024 dx  115 (114)        139 (145)     232 (225)
//   32768, 2048, 1024 dw  118 (125), 8     127 (139), 4  241 (209)   and K in 8 or 4 splits
//   4096, 1024, 1024 fwd  29 (34)          13.5 (13.2)   18 (18)
//   2048, 1024, 512 fwd   18 (22)          9.0 (9.5)     7.3 (7.3)
//   512, 4096, 4096 fwd   38 (45), 4       29 (28), 2    35 (30)
// The largest tile runs x w^T of 32768 x 2048 x 1024 at 0.97 PFLOP/s with warm caches and at
// 0.80 where y goes to memory (172 us): all CUs store their tiles at the same time, and no
// registers are left to hold a tile back and store it during the next one's slices.
double tile_us(int M, int N, int K, int T, int split) {
  const double slice = T == 256 ? 0.76 : T == 128 ? 0.235 : 0.1, ends = T == 256 ? 7.0 : T == 128 ? 2.7 : 0.55;
  const int64_t slices = ((K + split - 1) / split + BK - 1) / BK, per_cu = (tiles_of(M, N, T) * split + 255) / 256;
  return 3.0 + per_cu * (slices * slice + ends) + (split > 1 ? 3.0 + 8e-6 * split * M * N / 9.0 : 0.0);
}

int pick_tile(int M, int N, int K, int split, bool direct) {
  int best = 64;
  for (int T : kTileSizes)
    if ((T < 256 || direct) && tile_us(M, N, K, T, split) < tile_us(M, N, K, best, split)) best = T;
  return best;
}

// Whether an operand's rows are whole 16-byte granules (pads: because zeros follow them
// up to one): its tile can go straight to LDS.
bool direct_ok(const void* p, int64_t ld, int64_t extent, bool kc, bool pads) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0 && (extent % 8 == 0 || pads) &&
         (kc ? 256 * ld + 64 : 64 * ld + 256) < (int64_t(1) << 29);
}

typedef void (*GemmBf16Fn)(GemmBf16Args);

template <int LAYOUT, int BT, int WJ, bool DIRECT>
GemmBf16Fn pick(bool part) {
  if constexpr (LAYOUT == kGemmTN)
    return gemm_bf16_kernel<BT, WJ, LAYOUT, DIRECT, kEither>;
  else
    return part ? gemm_bf16_kernel<BT, WJ, LAYOUT, DIRECT, kSums> : gemm_bf16_kernel<BT, WJ, LAYOUT, DIRECT, kOutputs>;
}

template <int LAYOUT>
GemmBf16Fn kernel_of(int T, bool direct, bool part) {
  if (T == 256) return pick<LAYOUT, 256, 4, true>(part);
  if (T == 128) return direct ? pick<LAYOUT, 128, 2, true>(part) : pick<LAYOUT, 128, 2, false>(part);
  return direct ? pick<LAYOUT, 64, 2, true>(part) : pick<LAYOUT, 64, 2, false>(part);
}

}  // namespace

// Rows of M at most 32 straight from memory, unless K is long (a wave's turns of it come one
// after the other, where tiles split K) or w is wide (tiles read each of its lines once and
// in order). Measured in us, straight and in tiles, w in cache:
//   8, 2048, 1024    4.8  6.4   32, 2048, 1024  5.4  6.7   8, 1811, 1001  6.1 18.9
//   8, 2048, 2048    5.4  7.1   32, 2048, 2048  7.7  8.0   32, 1001, 4003 31.0 17.8
//   8, 2048, 4096    8.4  8.0   32, 2048, 4096 13.9  9.1
//   8, 8192, 1024    5.4  6.4   32, 4096, 1024  5.2  6.7
//   8, 16384, 1024   9.1  7.6   32, 8192, 1024  7.7  6.7
bool gemm_bf16_few_rows(int M, int N, int K) { return M <= 32 && K <= 2048 && N <= (M <= 16 ? 8192 : 4096); }

int gemm_bf16_pick_split(int M, int N, int K) {
  int best = 1;
  double least = 1e30;
  for (int split = 1; split <= 32 && (split == 1 || K / split >= 4 * BK); split *= 2)
    for (int T : kTileSizes) {
      const double us = tile_us(M, N, K, T, split);
      if (us < least) {
        least = us;
        best = split;
      }
    }
  return best;
}

namespace {

int check(const GemmBf16Args& g, const char* who) {
  if (g.M < 1 || g.N < 1 || g.K < 1 || g.ksplit < 1 || g.ksplit > 32 || (g.ksplit & (g.ksplit - 1)) != 0)
    return set_error(GS_ERR_INVALID, "%s: GEMM dims must be positive and ksplit a power of 2 (M=%d, N=%d, K=%d, ksplit=%d)",
                     who, g.M, g.N, g.K, g.ksplit);
  return GS_OK;
}

bool direct_of(const GemmBf16Args& g) {
  const bool a_kc = g.layout != kGemmTN, b_kc = g.layout == kGemmNT;
  return direct_ok(g.a, g.lda, a_kc ? g.K : g.M, a_kc, g.a_pads) && direct_ok(g.b, g.ldb, b_kc ? g.K : g.N, b_kc, g.b_pads);
}

// Workgroups of a product in tiles of T: a multiple of 8.
int64_t groups_of(const GemmBf16Args& g, int T) {
  const int64_t tiles = tiles_of(g.M, g.N, T), spread = g.ksplit < 8 ? 8 / g.ksplit : 1;
  return 8 * ((tiles + spread - 1) / spread) * (g.ksplit < 8 ? 1 : (g.ksplit + 7) / 8);
}

int finish(const GemmBf16Args& g, hipStream_t stream) {
  const int64_t octets = (int64_t)g.M * ((g.N + 7) / 8);
  hipLaunchKernelGGL(gemm_bf16_finish_kernel, dim3((unsigned)std::min<int64_t>((octets + 255) / 256, 8192)), dim3(256), 0,
                     stream, g);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}

constexpr int64_t kMostGroups = 1 << 22;

}  // namespace

int gemm_bf16(const GemmBf16Args& g, hipStream_t stream, const char* who) {
  const int rc = check(g, who);
  if (rc) return rc;
  if (g.layout == kGemmNT && g.ksplit == 1 && gemm_bf16_few_rows(g.M, g.N, g.K)) {
    hipLaunchKernelGGL(g.M <= 16 ? gemm_bf16_rows_kernel<1> : gemm_bf16_rows_kernel<2>, dim3((unsigned)((g.N + 15) / 16)),
                       dim3(64 * kRowWaves), 0, stream, g);
    GS_CHECK_HIP(hipGetLastError());
    return GS_OK;
  }
  const bool direct = direct_of(g), part = g.ksplit > 1;
  const int T = pick_tile(g.M, g.N, g.K, g.ksplit, direct);
  GemmBf16Fn fn = g.layout == kGemmNT   ? kernel_of<kGemmNT>(T, direct, part)
                  : g.layout == kGemmNN ? kernel_of<kGemmNN>(T, direct, part)
                                        : kernel_of<kGemmTN>(T, direct, part);
  const int64_t groups = groups_of(g, T);
  if (groups > kMostGroups) return set_error(GS_ERR_INVALID, "%s: GEMM of too many tiles (M=%d, N=%d)", who, g.M, g.N);
  hipLaunchKernelGGL(fn, dim3((unsigned)groups), dim3(T == 256 ? 512 : 256), 0, stream, g);
  GS_CHECK_HIP(hipGetLastError());
  return part ? finish(g, stream) : GS_OK;
}

bool gemm_bf16_pair_applies(const GemmBf16Args& x, const GemmBf16Args& w) {
  const bool direct = direct_of(x);
  return x.ksplit == 1 && direct == direct_of(w) && pick_tile(x.M, x.N, x.K, x.ksplit, direct) == 64 &&
         pick_tile(w.M, w.N, w.K, w.ksplit, direct) == 64 && groups_of(x, 64) + groups_of(w, 64) <= kMostGroups;
}

int gemm_bf16_pair(const GemmBf16Args& x, const GemmBf16Args& w, const ColumnSums& c, hipStream_t stream, const char* who) {
  int rc = check(x, who);
  if (!rc) rc = check(w, who);
  if (rc) return rc;
  const bool direct = direct_of(x), part = w.ksplit > 1;
  const int nx = (int)groups_of(x, 64), nw = (int)groups_of(w, 64), nc = c.dst ? (c.n + 15) / 16 : 0;
  auto fn = direct ? gemm_bf16_pair_kernel<true> : gemm_bf16_pair_kernel<false>;
  hipLaunchKernelGGL(fn, dim3((unsigned)(nx + nw + nc)), dim3(256), 0, stream, x, w, c, nx, nw);
  GS_CHECK_HIP(hipGetLastError());
  return part ? finish(w, stream) : GS_OK;
}

}  // namespace gs
