// Embedding (gfx950): out[m] = scale w[token[m]], and the weight's gradient
//   dw[v] = scale sum over the m with token[m] = v of dout[m],
// all of dw written (zeros where a token does not occur). A negative token marks padding: its row
// of out is zero and it sends no gradient; one of V or more gives NaN and sends none.
//
// Bound by memory: rows of w, out and dout, once each, and dw. For the gradient the positions m are
// brought into lists by token: counted (a position's place in its list is what the counter held),
// given room, and put down; the order within a list depends on timing until the sum sorts it, so that
// results do not. A wave sorts a list of 16 or fewer by counting smaller ones, lane by lane, and
// sums its rows in that order. Longer lists are cut into chunks, a workgroup each, whose waves take a
// quarter of its rows; a list's order there comes from counting smaller ones too or, where it is long, from a bit
// for every position of a window. Windows of positions are counted one after the other, so that a list holds
// them in order and a chunk reads its own windows alone: an entry is read by the chunks of its window, 512 at most and
// 64 from 2^20 positions on, however long its list is. The chunks' sums are joined in order. 16384 tokens of
// 32000 x 1024 bf16: forward 10 us; backward 10 to count, 8 to give room, put down and clear, 18 for the sums (5.5 TB/s), 4 to join.
#include "gs_seq.h"

namespace gs {
namespace {

typedef unsigned int u4v __attribute__((ext_vector_type(4)));

struct EmbedParams {
  const void* tokens;
  const void* w;      // forward
  void* out;
  const void* dout;   // backward
  void* dw;
  float scale;
  int64_t M, so;      // rows, and the stride of out or dout
  int V, K, wide;     // wide: tokens of 64 bits
  // backward: scratch
  uint32_t *count, *start, *place, *list;  // [V], [V], [M], [M]
  uint32_t* cursor;                        // room taken, chunks, rows of sums
  uint4* chunks;                           // token, first row of its sums, chunk, chunks of the token
  float* sums;                             // [rows][K]: of the chunks of lists that have several
  int chunk, most_chunks;
};

__device__ __forceinline__ int64_t token_at(const EmbedParams& p, int64_t m) {
  return p.wide ? static_cast<const int64_t*>(p.tokens)[m] : static_cast<const int32_t*>(p.tokens)[m];
}

// 16 bytes a lane, or one element where rows are not aligned to that.
template <typename T, bool VEC>
struct Row {
  static constexpr int kElems = VEC ? 16 / (int)sizeof(T) : 1;
  struct Raw {
    unsigned int w[VEC ? 4 : 1];
  };
  static __device__ __forceinline__ Raw load(const T* src) {
    Raw r;
    if constexpr (VEC) {
      const u4v q = *reinterpret_cast<const u4v*>(src);
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[i] = q[i];
    } else {
      r.w[0] = sizeof(T) == 2 ? *reinterpret_cast<const unsigned short*>(src) : *reinterpret_cast<const unsigned int*>(src);
    }
    return r;
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&x)[kElems]) {
    if constexpr (!VEC) {
      x[0] = Elem<T>::value(r.w[0]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
          x[2 * i] = __uint_as_float(r.w[i] << 16);
          x[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
        } else {
          x[i] = __uint_as_float(r.w[i]);
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

// A wave a row.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(EmbedParams p) {
  typedef Row<T, VEC> R;
  const int lane = threadIdx.x & 63;
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= p.M) return;
  const int64_t v = token_at(p, m);
  T* out = static_cast<T*>(p.out) + m * p.so;
  const T* w = static_cast<const T*>(p.w) + (v >= 0 && v < p.V ? v : 0) * p.K;
  for (int k = lane * R::kElems; k < p.K; k += 64 * R::kElems) {
    float x[R::kElems];
    if (v >= 0 && v < p.V) {
      R::unpack(R::load(w + k), x);
#pragma unroll
      for (int i = 0; i < R::kElems; ++i) x[i] *= p.scale;
    } else {
#pragma unroll
      for (int i = 0; i < R::kElems; ++i) x[i] = v < 0 ? 0.0f : __builtin_nanf("");
    }
    R::store(out + k, x);
  }
}

__global__ __launch_bounds__(256) void embed_clear_kernel(uint32_t* p, int64_t n) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e < n) p[e] = 0;
}

constexpr int kWindow = 1 << 17;  // positions that are counted, and ordered, at a time

// The window of positions from `from` on. Equal tokens of a wave are counted together, in one access: those of a
// frequent token would wait for each other (16384 tokens, one in 15 the same: 15 -> 10 us).
__global__ __launch_bounds__(256) void embed_count_kernel(EmbedParams p, int64_t from) {
  const int64_t m = from + (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t token = m < p.M ? token_at(p, m) : -1;
  const bool some = token >= 0 && token < p.V;
  const int v = (int)token, lane = threadIdx.x & 63;
  uint64_t left = __builtin_amdgcn_ballot_w64(some);
  int leader = lane, before = 0, count = 0;
  while (left) {  // uniform: once for each token of the wave
    const int l = __builtin_ctzll(left);
    const uint64_t same = __builtin_amdgcn_ballot_w64(some && v == __builtin_amdgcn_readlane(v, l));
    if (same >> lane & 1) {
      leader = l;
      before = __popcll(same & ((uint64_t(1) << lane) - 1));
      count = __popcll(same);
    }
    left &= ~same;
  }
  uint32_t base = 0;
  if (some && leader == lane) base = atomicAdd(p.count + v, (uint32_t)count);
  base = __shfl(base, leader);
  if (some) p.place[m] = base + before;
}

// Positions of a list that a wave sums. A step of 16384 tokens of 32000 x 1024 bf16, of 1237 of 1003 x 333 fp32 and
// of 30000 of 3000 x 512 bf16 takes 54, 25 and 55 us with 4, 53, 24 and 55 with 16, 61, 30 and 74 with 64.
constexpr uint32_t kShort = 16;

// What a list of n positions takes up: room, chunks where it is long, and a row for the sums of each of several chunks.
struct Needs {
  uint32_t x[3];
  __device__ __forceinline__ Needs(const EmbedParams& p, uint32_t n) {
    x[0] = n;
    x[1] = n > kShort ? (n + p.chunk - 1) / p.chunk : 0;
    x[2] = x[1] > 1 ? x[1] : 0;
  }
};
// The needs of the wave's lanes up to this one.
__device__ __forceinline__ void sum_up(Needs& a) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t o = __shfl_up(a.x[k], d);
      if (lane >= d) a.x[k] += o;
    }
  }
}
__device__ __forceinline__ void put_chunks(const EmbedParams& p, uint32_t v, uint32_t parts, uint32_t first, uint32_t row) {
  for (uint32_t c = 0; c < parts && first + c < (uint32_t)p.most_chunks; ++c) p.chunks[first + c] = uint4{v, row, c, parts};
}

// Room for each token's list, in no particular order, and the chunks of the long ones.
__global__ __launch_bounds__(1024) void embed_room_kernel(EmbedParams p) {
  __shared__ uint32_t waves[3][16], base[3];
  const int v = blockIdx.x * 1024 + threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Needs mine(p, v < p.V ? p.count[v] : 0);
  Needs upto = mine;
  sum_up(upto);
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (lane == 63) waves[k][wave] = upto.x[k];
  __syncthreads();
  if (threadIdx.x < 3) {
    uint32_t all = 0;
    for (int w = 0; w < 16; ++w) {
      const uint32_t x = waves[threadIdx.x][w];
      waves[threadIdx.x][w] = all;
      all += x;
    }
    base[threadIdx.x] = all ? atomicAdd(p.cursor + threadIdx.x, all) : 0;
  }
  __syncthreads();
  uint32_t at[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) at[k] = base[k] + waves[k][wave] + upto.x[k] - mine.x[k];
  if (mine.x[0]) p.start[v] = at[0];
  put_chunks(p, (uint32_t)v, mine.x[1], at[1], at[2]);
}

__global__ __launch_bounds__(256) void embed_place_kernel(EmbedParams p) {
  const int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (m >= p.M) return;
  const int64_t v = token_at(p, m);
  if (v >= 0 && v < p.V) p.list[p.start[v] + p.place[m]] = (uint32_t)m;
}

// All of the lists by one workgroup, whose counters are in LDS, where tokens are few: one launch instead of
// four (1237 tokens of 1003: 14 -> 4.6 us on the GPU; 16384 of 32000 would take 61, four launches 19).
constexpr int kOneTokens = 4096, kOneVocabulary = 4096;
__global__ __launch_bounds__(1024) void embed_lists_kernel(EmbedParams p) {
  constexpr int kEach = kOneTokens / 1024;
  __shared__ uint32_t count[kOneVocabulary];
  __shared__ uint32_t waves[3][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int v = threadIdx.x; v < p.V; v += 1024) count[v] = 0;
  int token[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int64_t m = i * 1024 + (int64_t)threadIdx.x, t = m < p.M ? token_at(p, m) : -1;
    token[i] = t >= 0 && t < p.V ? (int)t : -1;
  }
  __syncthreads();
  uint32_t place[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) place[i] = token[i] >= 0 ? atomicAdd(count + token[i], 1u) : 0;
  __syncthreads();
  // room: a thread takes `per` tokens; then the room of the threads before it
  const int per = (p.V + 1023) / 1024, v0 = threadIdx.x * per;
  Needs mine(p, 0);
  for (int v = v0; v < min(v0 + per, p.V); ++v) {
    const Needs one(p, count[v]);
#pragma unroll
    for (int k = 0; k < 3; ++k) mine.x[k] += one.x[k];
  }
  Needs upto = mine;
  sum_up(upto);
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (lane == 63) waves[k][wave] = upto.x[k];
  __syncthreads();
  if (threadIdx.x < 3) {
    uint32_t all = 0;
    for (int w = 0; w < 16; ++w) {
      const uint32_t x = waves[threadIdx.x][w];
      waves[threadIdx.x][w] = all;
      all += x;
    }
    p.cursor[threadIdx.x] = all;
  }
  __syncthreads();
  uint32_t at[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) at[k] = waves[k][wave] + upto.x[k] - mine.x[k];
  for (int v = v0; v < min(v0 + per, p.V); ++v) {
    const uint32_t n = count[v];
    const Needs one(p, n);
    p.count[v] = n;
    p.start[v] = count[v] = at[0];
    put_chunks(p, (uint32_t)v, one.x[1], at[1], at[2]);
#pragma unroll
    for (int k = 0; k < 3; ++k) at[k] += one.x[k];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (token[i] >= 0) p.list[count[token[i]] + place[i]] = (uint32_t)(i * 1024 + threadIdx.x);
}

// What a wave sums at once: kCols elements of a lane, of columns from k on, in rows whose loads are in flight together.
template <typename T, bool VEC>
struct Sum {
  typedef Row<T, VEC> R;
  static constexpr int kCols = VEC ? 2 : 8, kRows = 4, kSpan = 64 * R::kElems * kCols;
  float s[kCols][R::kElems];
  // rows row(0) .. row(n - 1) of dout, in that order (row: uniform)
  template <typename F>
  __device__ __forceinline__ void rows(const EmbedParams& p, int n, int k, F&& row) {
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int i = 0; i < R::kElems; ++i) s[c][i] = 0.0f;
    const T* dout = static_cast<const T*>(p.dout);
    for (int j0 = 0; j0 < n; j0 += kRows) {
      typename R::Raw raw[kRows][kCols];
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        if (j0 + j >= n) break;  // uniform
        const T* src = dout + (int64_t)row(j0 + j) * p.so;
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          if (k + c * 64 * R::kElems < p.K) raw[j][c] = R::load(src + k + c * 64 * R::kElems);
      }
#pragma unroll
      for (int j = 0; j < kRows; ++j) {
        if (j0 + j >= n) break;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          if (k + c * 64 * R::kElems >= p.K) continue;
          float x[R::kElems];
          R::unpack(raw[j][c], x);
#pragma unroll
          for (int i = 0; i < R::kElems; ++i) s[c][i] += x[i];
        }
      }
    }
  }
  __device__ __forceinline__ void store(const EmbedParams& p, int64_t v, int k) {
    T* dw = static_cast<T*>(p.dw) + v * p.K;
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      if (k + c * 64 * R::kElems >= p.K) continue;
      float x[R::kElems];
#pragma unroll
      for (int i = 0; i < R::kElems; ++i) x[i] = s[c][i] * p.scale;
      R::store(dw + k + c * 64 * R::kElems, x);
    }
  }
};

// A workgroup a chunk of a long list: the positions of ranks chunk c to chunk (c + 1). With kAll
// positions or fewer, a rank is counted; otherwise bits of a window's positions say which are in
// the list, and those before one, with the windows before, are its rank.
constexpr int kMostChunk = 2048, kAll = 256, kMostSpan = 1024;
union ChunkShared {
  struct {
    uint32_t bits[kWindow / 32], upto[256];
  } sort;
  uint32_t all[kAll];
  float sums[3][kMostSpan];
};

template <typename T, bool VEC>
__device__ __forceinline__ void sum_chunk(const EmbedParams& p, const uint4 c, ChunkShared& lds, uint32_t* rows) {
  typedef Sum<T, VEC> S;
  static_assert(S::kSpan <= kMostSpan, "columns of a pass");
  const uint32_t n = p.count[c.x], from = c.z * p.chunk, to = min(n, from + p.chunk);
  const uint32_t* list = p.list + p.start[c.x];
  if (n <= kAll) {
    const uint32_t mine = threadIdx.x < n ? list[threadIdx.x] : 0xffffffffu;
    lds.all[threadIdx.x] = mine;
    __syncthreads();
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += lds.all[j] < mine ? 1 : 0;
    if (threadIdx.x < n && rank >= from && rank < to) rows[rank - from] = mine;
  } else {
    // the end of the window that entry i is in, of entries i to i + kWindow (no more than that are in one), or its start
    auto edge = [&](uint32_t i, bool end) {
      if (p.M <= kWindow) return end ? n : 0u;
      const uint32_t w = list[i] / kWindow;
      uint32_t lo = end ? i : i - min(i, (uint32_t)kWindow), hi = end ? (uint32_t)min((int64_t)n, (int64_t)i + kWindow) : i;
      while (lo < hi) {  // the first entry in [lo, hi) of a window behind w, or of w, or hi
        const uint32_t mid = lo + (hi - lo) / 2, v = list[mid] / kWindow;
        if (end ? v > w : v >= w) hi = mid;
        else lo = mid + 1;
      }
      return lo;
    };
    for (uint32_t first = edge(from, false), last; first < to; first = last) {
      last = edge(first, true);
      const int64_t base = (int64_t)(list[first] / kWindow) * kWindow;
      const int words = (int)min((int64_t)kWindow, p.M - base + 31) / 32;
      for (int i = threadIdx.x; i < words; i += 256) lds.sort.bits[i] = 0;
      __syncthreads();
      for (uint32_t i = first + threadIdx.x; i < last; i += 256) {
        const uint32_t at = list[i] - (uint32_t)base;
        if (at < (uint32_t)kWindow) atomicOr(lds.sort.bits + at / 32, 1u << (at & 31));
      }
      __syncthreads();
      // each thread counts the bits of a run of words; then the runs before it
      const int per = (words + 255) / 256, w0 = threadIdx.x * per;
      uint32_t mine = 0;
      for (int i = w0; i < min(w0 + per, words); ++i) mine += __popc(lds.sort.bits[i]);
      lds.sort.upto[threadIdx.x] = mine;
      __syncthreads();
      for (int d = 1; d < 256; d *= 2) {
        const uint32_t o = (int)threadIdx.x >= d ? lds.sort.upto[threadIdx.x - d] : 0;
        __syncthreads();
        lds.sort.upto[threadIdx.x] += o;
        __syncthreads();
      }
      uint32_t rank = first + lds.sort.upto[threadIdx.x] - mine;
      if (rank < to && rank + mine > from) {
        for (int i = w0; i < min(w0 + per, words); ++i)
          for (uint32_t w = lds.sort.bits[i]; w; w &= w - 1, ++rank)
            if (rank >= from && rank < to) rows[rank - from] = (uint32_t)(base + 32 * i + __ffs(w) - 1);
      }
      __syncthreads();
    }
  }
  // a quarter of the rows a wave, joined in order
  const int count = (int)(to - from), quarter = (count + 3) / 4, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), first = min(count, wave * quarter);
  const int mine = min(count, first + quarter) - first;
  for (int k0 = 0; k0 < p.K; k0 += S::kSpan) {
    const int k = k0 + lane * S::R::kElems;
    __syncthreads();
    S sum;
    sum.rows(p, mine, k, [&](int j) { return __builtin_amdgcn_readfirstlane(rows[first + j]); });
    if (wave > 0) {
#pragma unroll
      for (int e = 0; e < S::kCols; ++e)
#pragma unroll
        for (int i = 0; i < S::R::kElems; ++i) lds.sums[wave - 1][(e * S::R::kElems + i) * 64 + lane] = sum.s[e][i];
    }
    __syncthreads();
    if (wave != 0) continue;
#pragma unroll
    for (int e = 0; e < S::kCols; ++e)
#pragma unroll
      for (int i = 0; i < S::R::kElems; ++i) {
        float& x = sum.s[e][i];
#pragma unroll
        for (int w = 0; w < 3; ++w) x += lds.sums[w][(e * S::R::kElems + i) * 64 + lane];
        const int at = k + e * 64 * S::R::kElems + i;
        if (c.w > 1 && at < p.K) p.sums[((int64_t)c.y + c.z) * p.K + at] = x;
      }
    if (c.w == 1) sum.store(p, c.x, k);
  }
}

// The first workgroups take a chunk of a long list each; a wave of the others four tokens
// whose lists are short or empty.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedParams p) {
  typedef Sum<T, VEC> S;
  __shared__ ChunkShared lds;
  __shared__ uint32_t rows[kMostChunk];
  if ((int)blockIdx.x < p.most_chunks) {  // uniform
    if (blockIdx.x < p.cursor[1]) sum_chunk<T, VEC>(p, p.chunks[blockIdx.x], lds, rows);
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int v0 = ((int)(blockIdx.x - p.most_chunks) * 4 + wave) * 4;
  const bool some = lane < 4 && v0 + lane < p.V;
  const int counts = some ? (int)p.count[v0 + lane] : -1;
  const int starts = counts > 0 ? (int)p.start[v0 + lane] : 0;
  int list[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int n = __builtin_amdgcn_readlane(counts, t);
    list[t] = lane < n && n <= (int)kShort ? (int)p.list[(uint32_t)__builtin_amdgcn_readlane(starts, t) + lane] : 0x7fffffff;
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int n = __builtin_amdgcn_readlane(counts, t);
    if (n < 0 || n > (int)kShort) continue;
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += __builtin_amdgcn_readlane(list[t], j) < list[t] ? 1 : 0;
    // lane r gets the position of rank r (lanes without one send theirs past the list)
    const int sorted = __builtin_amdgcn_ds_permute(4 * (lane < n ? rank : lane), list[t]);
    for (int k0 = 0; k0 < p.K; k0 += S::kSpan) {
      const int k = k0 + lane * S::R::kElems;
      S sum;
      sum.rows(p, n, k, [&](int j) { return __builtin_amdgcn_readlane(sorted, j); });
      sum.store(p, v0 + t, k);
    }
  }
}

// The chunks of a list of several in order: a workgroup a chunk, of which the first of each list works.
template <typename T>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedParams p) {
  if (blockIdx.x >= min(p.cursor[1], (uint32_t)p.most_chunks)) return;
  const uint4 c = p.chunks[blockIdx.x];
  if (c.z != 0 || c.w == 1) return;
  for (int k = blockIdx.y * 256 + threadIdx.x; k < p.K; k += gridDim.y * 256) {
    const float* src = p.sums + (int64_t)c.y * p.K + k;
    float s = 0.0f;
    for (uint32_t j0 = 0; j0 < c.w; j0 += 8) {
      float x[8];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) x[j] = j0 + j < c.w ? src[(int64_t)(j0 + j) * p.K] : 0.0f;
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j)
        if (j0 + j < c.w) s += x[j];
    }
    static_cast<T*>(p.dw)[(int64_t)c.x * p.K + k] = (T)(s * p.scale);
  }
}

// ---- host ---------------------------------------------------------------------------

struct Plan {
  int chunk, most_chunks;
  int64_t start, place, list, chunks, sums, total, clear;  // offsets; words to clear from the start
};
// Chunks of 64 positions, longer ones where there are more than 2^15 (a chunk reads the whole list).
Plan make_plan(int64_t M, int64_t V, int64_t K) {
  Plan r;
  r.chunk = (int)std::min<int64_t>(kMostChunk, std::max<int64_t>(64, (M / 512 + 63) / 64 * 64));
  // a list of n > kShort has n / chunk rounded up
  r.most_chunks = M > kShort ? (int)(M / r.chunk + std::min<int64_t>(V, M / (kShort + 1))) : 0;
  // and, of n > chunk, less than 2 n / chunk, each with a row of sums
  const int64_t rows = M > r.chunk ? 2 * M / r.chunk : 0;
  r.clear = 64 + V;  // cursors on a line of their own, counts
  r.start = align256(r.clear * 4);
  r.place = r.start + align256(V * 4);
  r.list = r.place + align256(M * 4);
  r.chunks = r.list + align256(M * 4);
  r.sums = r.chunks + align256((int64_t)r.most_chunks * 16);
  r.total = r.sums + align256(rows * K * 4);
  return r;
}

template <typename Args>
int check(const Args* a, const char* who, int64_t stride) {
  if (a == nullptr) return set_error(GS_ERR_INVALID, "%s: args is NULL", who);
  if (a->M < 1 || a->V < 1 || a->K < 1)
    return set_error(GS_ERR_INVALID, "%s: M, V and K must be > 0; got M=%lld, V=%lld, K=%lld", who, (long long)a->M,
                     (long long)a->V, (long long)a->K);
  if (a->M > (1ll << 25) || a->V > (1ll << 25) || a->K > (1ll << 20))
    return set_error(GS_ERR_INVALID, "%s: M/V/K out of supported range (M=%lld, V=%lld, K=%lld)", who, (long long)a->M,
                     (long long)a->V, (long long)a->K);
  if (a->token_bits != 32 && a->token_bits != 64)
    return set_error(GS_ERR_INVALID, "%s: tokens must have 32 or 64 bits; got %d", who, a->token_bits);
  if (!(std::isfinite(a->scale))) return set_error(GS_ERR_INVALID, "%s: scale must be finite; got %g", who, (double)a->scale);
  if (a->M > 1 && stride < a->K)
    return set_error(GS_ERR_INVALID, "%s: a row stride of %lld does not hold K=%lld", who, (long long)stride, (long long)a->K);
  return check_dtype(who, a->dtype);
}

int make_lists(const EmbedParams& p, const Plan& plan, hipStream_t stream) {
  const dim3 rows((unsigned)((p.M + 255) / 256));
  hipLaunchKernelGGL(embed_clear_kernel, dim3((unsigned)((plan.clear + 255) / 256)), dim3(256), 0, stream, p.cursor, plan.clear);
  GS_CHECK_HIP(hipGetLastError());
  for (int64_t from = 0; from < p.M; from += kWindow) {
    const int64_t n = std::min<int64_t>(kWindow, p.M - from);
    hipLaunchKernelGGL(embed_count_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p, from);
    GS_CHECK_HIP(hipGetLastError());
  }
  hipLaunchKernelGGL(embed_room_kernel, dim3((unsigned)((p.V + 1023) / 1024)), dim3(1024), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  hipLaunchKernelGGL(embed_place_kernel, rows, dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}

bool aligned16(const void* p, int64_t stride, int size) {
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride * size % 16 == 0;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_embedding_fwd(const gs_embedding_args* a, hipStream_t stream) {
  const char* who = "gs_embedding_fwd";
  clear_error();
  const int rc = check(a, who, a ? a->so : 0);
  if (rc) return rc;
  if (!a->tokens || !a->w || !a->out)
    return set_error(GS_ERR_INVALID, "%s: tokens, w and out must be non-NULL device pointers", who);
  const int size = a->dtype == GS_DTYPE_F32 ? 4 : 2;
  EmbedParams p{};
  p.tokens = a->tokens;
  p.w = a->w;
  p.out = a->out;
  p.scale = a->scale;
  p.M = a->M;
  p.so = a->so;
  p.V = (int)a->V;
  p.K = (int)a->K;
  p.wide = a->token_bits == 64;
  const bool vec = aligned16(a->w, a->K, size) && aligned16(a->out, a->so, size);
  auto fn = size == 4 ? (vec ? embed_fwd_kernel<float, true> : embed_fwd_kernel<float, false>)
                      : (vec ? embed_fwd_kernel<__bf16, true> : embed_fwd_kernel<__bf16, false>);
  hipLaunchKernelGGL(fn, dim3((unsigned)((a->M + 3) / 4)), dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  return GS_OK;
}

extern "C" int64_t gs_embedding_bwd_scratch_bytes(const gs_embedding_bwd_args* a) {
  const char* who = "gs_embedding_bwd_scratch_bytes";
  clear_error();
  const int rc = check(a, who, a ? a->sdo : 0);
  return rc ? rc : make_plan(a->M, a->V, a->K).total;
}

extern "C" int gs_embedding_bwd(const gs_embedding_bwd_args* a, hipStream_t stream) {
  const char* who = "gs_embedding_bwd";
  clear_error();
  int rc = check(a, who, a ? a->sdo : 0);
  if (rc) return rc;
  if (!a->tokens || !a->dout || !a->dw)
    return set_error(GS_ERR_INVALID, "%s: tokens, dout and dw must be non-NULL device pointers", who);
  const Plan plan = make_plan(a->M, a->V, a->K);
  if ((rc = check_plain_scratch(who, a->scratch, a->scratch_bytes, plan.total))) return rc;
  const int size = a->dtype == GS_DTYPE_F32 ? 4 : 2;
  char* s = static_cast<char*>(a->scratch);
  EmbedParams p{};
  p.tokens = a->tokens;
  p.dout = a->dout;
  p.dw = a->dw;
  p.scale = a->scale;
  p.M = a->M;
  p.so = a->sdo;
  p.V = (int)a->V;
  p.K = (int)a->K;
  p.wide = a->token_bits == 64;
  p.cursor = reinterpret_cast<uint32_t*>(s);
  p.count = p.cursor + 64;
  p.start = reinterpret_cast<uint32_t*>(s + plan.start);
  p.place = reinterpret_cast<uint32_t*>(s + plan.place);
  p.list = reinterpret_cast<uint32_t*>(s + plan.list);
  p.chunks = reinterpret_cast<uint4*>(s + plan.chunks);
  p.sums = reinterpret_cast<float*>(s + plan.sums);
  p.chunk = plan.chunk;
  p.most_chunks = plan.most_chunks;
  if (a->M <= kOneTokens && a->V <= kOneVocabulary) {
    hipLaunchKernelGGL(embed_lists_kernel, dim3(1), dim3(1024), 0, stream, p);
    GS_CHECK_HIP(hipGetLastError());
  } else {
    if ((rc = make_lists(p, plan, stream))) return rc;
  }
  const bool vec = aligned16(a->dw, a->K, size) && aligned16(a->dout, a->sdo, size);
  auto sum = size == 4 ? (vec ? embed_sum_kernel<float, true> : embed_sum_kernel<float, false>)
                       : (vec ? embed_sum_kernel<__bf16, true> : embed_sum_kernel<__bf16, false>);
  hipLaunchKernelGGL(sum, dim3((unsigned)(plan.most_chunks + (a->V + 15) / 16)), dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  if (a->M > plan.chunk) {  // there may be a list of several chunks
    hipLaunchKernelGGL(size == 4 ? embed_join_kernel<float> : embed_join_kernel<__bf16>, dim3((unsigned)plan.most_chunks, 4),
                       dim3(256), 0, stream, p);
    GS_CHECK_HIP(hipGetLastError());
  }
  return GS_OK;
}
