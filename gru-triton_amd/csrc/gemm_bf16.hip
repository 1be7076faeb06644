// bf16 products on v_mfma_f32_16x16x32_bf16 (gfx950) for the linear operator: x w^T
// (NT), dpre w (NN) and dpre^T x (TN), with the bias, activation and residual of the
// forward in the epilogue.
//
// A workgroup computes a BM x BN tile of C, K in slices of 64, double-buffered in LDS.
// The MFMA takes B's tile as its first operand, so that a lane holds four consecutive
// columns of one row of C (D VGPR v of lane l: C[l % 16][4 (l / 16) + v]) and stores
// them at once.
//
// LDS layouts (16-byte granules, no padding):
//   operand contiguous along k: row r is 8 granules of 8 k; granule c sits in slot
//     c ^ (r % 8). A lane reads k = 8 (l / 16) + 32 kk of row l % 16 in 16 bytes; the
//     16 lanes of a pass (rows r < 8 of one k-group and r >= 8 of another) then cover
//     all 64 banks.
//   operand contiguous along its rows: k-row k is R / 8 granules of 8 rows; granule g
//     sits in slot g ^ swz(k). ds_read_b64_tr_b16 gives lane l of each 16 four
//     consecutive k of row l % 16 (lane l supplies the address of k = l / 4, rows
//     4 (l % 4) .. + 3); the 8 k-rows that a pass of 32 lanes touches (k % 4 and bit 3
//     of k) sit in different 32-byte bank groups.
// Operands whose rows are 16-byte aligned come straight from memory to LDS
// (buffer_load ... lds, 16 bytes a lane; the swizzle is in the address each lane asks
// for, a lane past an edge asks for an offset out of range and gets zeros). Others go
// through registers, in 16-byte loads at any address, element by element where a
// granule crosses the end of a row.
#include "gs_gemm_bf16.h"

namespace gs {
namespace {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f2v __attribute__((ext_vector_type(2)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef unsigned int u2v __attribute__((ext_vector_type(2)));
typedef unsigned int u4v __attribute__((ext_vector_type(4)));
typedef unsigned int u4u __attribute__((ext_vector_type(4), aligned(2)));
typedef __attribute__((address_space(3))) void LdsVoid;
typedef __attribute__((address_space(3))) s4v LdsS4;

constexpr int BK = 64;

// One operand's tile of a slice: R rows x 64 k in LDS.
template <int R, bool KC, int THREADS>
struct Tile {
  static constexpr int kBytes = R * BK * 2, kWaves = THREADS / 64;
  static constexpr int kLoads = kBytes / 16 / THREADS;  // granules of a thread
  static_assert(kLoads >= 1, "a granule for every thread");

  static __device__ __forceinline__ int swz(int k) {
    return R >= 128 ? 2 * ((k & 3) | ((k >> 1) & 4)) : 2 * (((k >> 1) & 1) | ((k >> 2) & 2));
  }
  // row (the first of 8, if not KC) and k (the first of 8, if KC) of the granule at byte `at` of the tile
  static __device__ __forceinline__ void granule(int at, int* row, int* k) {
    if constexpr (KC) {
      *row = at >> 7;
      *k = (((at >> 4) & 7) ^ (*row & 7)) * 8;
    } else {
      *k = at / (2 * R);
      *row = (((at % (2 * R)) >> 4) ^ swz(*k)) * 8;
    }
  }

  // 16-byte fragment of MFMA step kk, rows row0 .. row0 + 15 (row0 a multiple of 16)
  static __device__ __forceinline__ bf8 fragment(const char* lds, int row0, int kk, int lane) {
    const int r = lane & 15, g = lane >> 4;
    if constexpr (KC) {
      const int at = (row0 + r) * 128 + (((4 * kk + g) ^ (r & 7)) << 4);
      return *reinterpret_cast<const bf8*>(lds + at);
    } else {
      const int k = 8 * g + (r >> 2);  // + 32 kk + 4 h: neither changes swz
      const int at = k * 2 * R + ((((row0 >> 3) + ((r & 3) >> 1)) ^ swz(k)) << 4) + ((r & 1) << 3) + kk * 64 * R;
      union {
        s4v h[2];
        bf8 v;
      } u;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsS4*)(lds + at + h * 8 * R));
      return u.v;
    }
  }
};

// Rows and k that exist: a load past them gives zeros.
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
    const uint32_t last = s == n - 1 ? ~0u : 0u;
    const auto r = bounded_rsrc(base + s * step, 0x7fffffffu);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int e = 0; e < T::kLoads; ++e)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (LdsVoid*)(lds + (wave * T::kLoads + e) * 1024), 16,
                                               (int)(off[e] | (tail[e] & last)), 0, 0, 0);
  }
};

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
  __device__ __forceinline__ void load(int s, u4v (&x)[T::kLoads]) const {
#pragma unroll
    for (int e = 0; e < T::kLoads; ++e) {
      int row, k;
      T::granule((threadIdx.x + e * THREADS) * 16, &row, &k);
      row += row0;
      k += kbeg + s * BK;
      // elements along the contiguous side that exist
      const int have = KC ? (row < lim ? kend - k : 0) : (k < kend ? lim - row : 0);
      const __bf16* q = p + (KC ? row * ld + k : k * ld + row);
      if (have >= 8) {
        x[e] = *reinterpret_cast<const u4u*>(q);
      } else {
        unsigned int w[4] = {0u, 0u, 0u, 0u};
        const unsigned short* h = reinterpret_cast<const unsigned short*>(q);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < have) w[i >> 1] |= (unsigned int)h[i] << (16 * (i & 1));
        x[e] = u4v{w[0], w[1], w[2], w[3]};
      }
    }
  }
  __device__ __forceinline__ void stage(char* lds, const u4v (&x)[T::kLoads]) const {
#pragma unroll
    for (int e = 0; e < T::kLoads; ++e)
      *reinterpret_cast<u4v*>(lds + (threadIdx.x + e * THREADS) * 16) = x[e];
  }
};

typedef unsigned int u2u __attribute__((ext_vector_type(2), aligned(2)));

// Four elements of a row from column j on, as far as they exist.
__device__ __forceinline__ void load_row4(const __bf16* p, int j, int N, float (&x)[4]) {
  if (j + 4 <= N) {
    const u2u w = *reinterpret_cast<const u2u*>(p + j);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = j + i < N ? (float)p[j + i] : 0.0f;
  }
}
__device__ __forceinline__ void store_row4(__bf16* p, int j, int N, const float (&x)[4]) {
  if (j + 4 <= N) {
    u2u w;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w[i] = __builtin_bit_cast(unsigned int, __builtin_convertvector((f2v{x[2 * i], x[2 * i + 1]}), bf2v));
    *reinterpret_cast<u2u*>(p + j) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i < N) p[j + i] = (__bf16)x[i];
  }
}

// What follows the sums of columns j .. j + 3 of row i (< M; columns from N on do not exist).
__device__ __forceinline__ void finish4(const LinearEpilogue& e, __bf16* y, int64_t ldy, int i, int j, int N,
                                        const float (&bias)[4], float (&x)[4]) {
#pragma unroll
  for (int v = 0; v < 4; ++v) x[v] += bias[v];
  if (e.pre != nullptr) store_row4(static_cast<__bf16*>(e.pre) + (int64_t)i * N, j, N, x);
  if (e.act != GS_ACT_NONE) {
#pragma unroll
    for (int v = 0; v < 4; ++v) x[v] = act_value(x[v], e.act);
  }
  if (e.residual != nullptr) {
    float r[4];
    load_row4(static_cast<const __bf16*>(e.residual) + i * e.ldr, j, N, r);
#pragma unroll
    for (int v = 0; v < 4; ++v) x[v] += r[v];
  }
  store_row4(y + i * ldy, j, N, x);
}

template <int BM, int BN, int WM, int WN, int LAYOUT, bool DIRECT, bool PART>
__global__ __launch_bounds__(64 * WM * WN, 2) void gemm_bf16_kernel(GemmBf16Args g) {
  constexpr int THREADS = 64 * WM * WN, TI = BM / WM / 16, TJ = BN / WN / 16;
  constexpr bool A_KC = LAYOUT != kGemmTN, B_KC = LAYOUT == kGemmNT;
  typedef typename std::conditional<DIRECT, Direct<BM, A_KC, THREADS>, Staged<BM, A_KC, THREADS>>::type LA;
  typedef typename std::conditional<DIRECT, Direct<BN, B_KC, THREADS>, Staged<BN, B_KC, THREADS>>::type LB;
  __shared__ __attribute__((aligned(1024))) char A0[LA::kBytes];
  __shared__ __attribute__((aligned(1024))) char A1[LA::kBytes];
  __shared__ __attribute__((aligned(1024))) char B0[LB::kBytes];
  __shared__ __attribute__((aligned(1024))) char B1[LB::kBytes];
  // Each XCD (workgroup mod 8) takes a run of tiles, in patches of 1024 rows.
  const int mt = (g.M + BM - 1) / BM, nt = (g.N + BN - 1) / BN, total = mt * nt, per = (total + 7) / 8;
  const int tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || tile >= total) return;  // uniform
  constexpr int kPatch = 1024 / BM;
  const int patch = tile / (kPatch * nt), in_patch = tile - patch * kPatch * nt;
  const int pm = min(kPatch, mt - patch * kPatch);
  const int i0 = (patch * kPatch + in_patch % pm) * BM, j0 = in_patch / pm * BN;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = (wave / WN) * TI * 16, wj = (wave % WN) * TJ * 16;
  const int kper = ((g.K + g.ksplit - 1) / g.ksplit + BK - 1) / BK * BK;
  const int kbeg = blockIdx.z * kper, kend = min(g.K, kbeg + kper);
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

  auto products = [&](const char* A, const char* B) __attribute__((always_inline)) {
#pragma unroll
    for (int kk = 0; kk < BK / 32; ++kk) {
      bf8 fa[TI], fb[TJ];
#pragma unroll
      for (int a = 0; a < TI; ++a) fa[a] = LA::fragment(A, wi + 16 * a, kk, lane);
#pragma unroll
      for (int b = 0; b < TJ; ++b) fb[b] = LB::fragment(B, wj + 16 * b, kk, lane);
#pragma unroll
      for (int a = 0; a < TI; ++a)
#pragma unroll
        for (int b = 0; b < TJ; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[b], fa[a], acc[a][b], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // A slice is read after the barrier that follows its arrival; the buffer it leaves is
  // filled again after the next one.
  if constexpr (DIRECT) {
    auto arrive = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    if (n > 0) {
      la.load(0, n, A0);
      lb.load(0, n, B0);
    }
    int s = 0;
    for (; s + 1 < n; s += 2) {  // in pairs, so that the loop has one exit
      arrive();
      la.load(s + 1, n, A1);
      lb.load(s + 1, n, B1);
      products(A0, B0);
      arrive();
      if (s + 2 < n) {
        la.load(s + 2, n, A0);
        lb.load(s + 2, n, B0);
      }
      products(A1, B1);
    }
    if (s < n) {
      arrive();
      products(A0, B0);
    }
  } else {
    u4v xa[LA::kLoads], xb[LB::kLoads];
    auto load = [&](int s) __attribute__((always_inline)) {
      la.load(s, xa);
      lb.load(s, xb);
    };
    auto stage = [&](char* A, char* B) __attribute__((always_inline)) {
      la.stage(A, xa);
      lb.stage(B, xb);
    };
    if (n > 0) {
      load(0);
      stage(A0, B0);
    }
    int s = 0;
    for (; s + 1 < n; s += 2) {
      lds_barrier();
      load(s + 1);
      products(A0, B0);
      stage(A1, B1);
      lds_barrier();
      if (s + 2 < n) load(s + 2);
      products(A1, B1);
      if (s + 2 < n) stage(A0, B0);
    }
    if (s < n) {
      lds_barrier();
      products(A0, B0);
    }
  }

  const int r16 = lane & 15, q4 = (lane >> 4) * 4;
#pragma unroll
  for (int b = 0; b < TJ; ++b) {
    const int j = j0 + wj + 16 * b + q4;
    if (j >= g.N) continue;
    float bias[4] = {0.f, 0.f, 0.f, 0.f};
    if (!PART && g.epi.bias != nullptr) load_row4(static_cast<const __bf16*>(g.epi.bias), j, g.N, bias);
#pragma unroll
    for (int a = 0; a < TI; ++a) {
      const int i = i0 + wi + 16 * a + r16;
      if (i >= g.M) continue;
      float x[4];
#pragma unroll
      for (int v = 0; v < 4; ++v) x[v] = acc[a][b][v];
      if constexpr (PART) {
        float* c = g.part + ((int64_t)blockIdx.z * g.M + i) * g.N + j;
        typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
        if (j + 4 <= g.N) {
          *reinterpret_cast<f4u*>(c) = f4u{x[0], x[1], x[2], x[3]};
        } else {
#pragma unroll
          for (int v = 0; v < 4; ++v)
            if (j + v < g.N) c[v] = x[v];
        }
      } else {
        finish4(g.epi, g.y, g.ldy, i, j, g.N, bias, x);
      }
    }
  }
}

// y from the splits' sums, added in order: four columns a thread.
__global__ __launch_bounds__(256) void gemm_bf16_finish_kernel(GemmBf16Args g) {
  const int quads = (g.N + 3) / 4;
  const int64_t all = (int64_t)g.M * quads;
  for (int64_t q = blockIdx.x * (int64_t)256 + threadIdx.x; q < all; q += (int64_t)gridDim.x * 256) {
    const int i = (int)(q / quads), j = (int)(q - (int64_t)i * quads) * 4;
    float x[4] = {0.f, 0.f, 0.f, 0.f}, bias[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < g.ksplit; ++s) {
      const float* c = g.part + ((int64_t)s * g.M + i) * g.N + j;
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (j + v < g.N) x[v] += c[v];
    }
    if (g.epi.bias != nullptr) load_row4(static_cast<const __bf16*>(g.epi.bias), j, g.N, bias);
    finish4(g.epi, g.y, g.ldy, i, j, g.N, bias, x);
  }
}

// ---- host ---------------------------------------------------------------------------

int64_t tiles_of(int M, int N, int T) { return (int64_t)((M + T - 1) / T) * ((N + T - 1) / T); }

int pick_tile(int M, int N, int ksplit) {
  if (tiles_of(M, N, 256) * ksplit >= 200) return 256;
  if (tiles_of(M, N, 128) * ksplit >= 200) return 128;
  return 64;
}

bool direct_ok(const void* p, int64_t ld, int64_t extent, bool kc) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0 && extent % 8 == 0 &&
         (kc ? 256 * ld + 64 : 64 * ld + 256) < (int64_t(1) << 29);
}

typedef void (*GemmBf16Fn)(GemmBf16Args);

template <int LAYOUT, int BT, int WM, int WN, bool DIRECT>
GemmBf16Fn pick(bool part) {
  return part ? gemm_bf16_kernel<BT, BT, WM, WN, LAYOUT, DIRECT, true> : gemm_bf16_kernel<BT, BT, WM, WN, LAYOUT, DIRECT, false>;
}

template <int LAYOUT>
GemmBf16Fn kernel_of(int T, bool direct, bool part) {
  if (T == 256) return pick<LAYOUT, 256, 2, 4, true>(part);
  if (T == 128) return direct ? pick<LAYOUT, 128, 2, 2, true>(part) : pick<LAYOUT, 128, 2, 2, false>(part);
  return direct ? pick<LAYOUT, 64, 2, 2, true>(part) : pick<LAYOUT, 64, 2, 2, false>(part);
}

}  // namespace

int gemm_bf16_pick_split(int M, int N, int K) {
  const int64_t tiles = tiles_of(M, N, 128);
  int s = 1;
  while (s < 32 && tiles * s < 256 && K / (s * 2) >= 256) s *= 2;
  return s;
}

int gemm_bf16(const GemmBf16Args& g, hipStream_t stream, const char* who) {
  if (g.M < 1 || g.N < 1 || g.K < 1 || g.ksplit < 1 || g.ksplit > 65535)
    return set_error(GS_ERR_INVALID, "%s: GEMM dims must be positive (M=%d, N=%d, K=%d, ksplit=%d)", who, g.M, g.N,
                     g.K, g.ksplit);
  const bool a_kc = g.layout != kGemmTN, b_kc = g.layout == kGemmNT;
  const bool direct = direct_ok(g.a, g.lda, a_kc ? g.K : g.M, a_kc) && direct_ok(g.b, g.ldb, b_kc ? g.K : g.N, b_kc);
  const int T = std::min(pick_tile(g.M, g.N, g.ksplit), direct ? 256 : 128);
  const bool part = g.ksplit > 1;
  GemmBf16Fn fn = g.layout == kGemmNT   ? kernel_of<kGemmNT>(T, direct, part)
                  : g.layout == kGemmNN ? kernel_of<kGemmNN>(T, direct, part)
                                        : kernel_of<kGemmTN>(T, direct, part);
  const int64_t tiles = 8 * ((tiles_of(g.M, g.N, T) + 7) / 8);
  if (tiles > (1 << 22)) return set_error(GS_ERR_INVALID, "%s: GEMM of too many tiles (M=%d, N=%d)", who, g.M, g.N);
  hipLaunchKernelGGL(fn, dim3((unsigned)tiles, 1, (unsigned)g.ksplit), dim3(T == 256 ? 512 : 256), 0, stream, g);
  GS_CHECK_HIP(hipGetLastError());
  if (part) {
    const int64_t quads = (int64_t)g.M * ((g.N + 3) / 4);
    hipLaunchKernelGGL(gemm_bf16_finish_kernel, dim3((unsigned)std::min<int64_t>((quads + 255) / 256, 4096)), dim3(256),
                       0, stream, g);
    GS_CHECK_HIP(hipGetLastError());
  }
  return GS_OK;
}

}  // namespace gs
