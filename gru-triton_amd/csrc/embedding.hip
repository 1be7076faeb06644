// Embedding (gfx950): out[m] = scale w[token[m]], and the weight's gradient
//   dw[v] = scale sum over the m with token[m] = v of dout[m],
// all of dw written (zeros where a token does not occur). A negative token marks padding: its row
// of out is zero and it sends no gradient; one of V or more gives NaN and sends none.
//
// Bound by memory: rows of w, out and dout, once each, and dw. For the gradient the positions m are
// brought into lists by token: counted (a position's place in its list is what the counter held),
// given room, and put down; the order within a list depends on timing until the sum sorts it, so that
// results do not. A wave sorts a list of 64 or fewer by counting smaller ones, lane by lane, and
// sums its rows in that order. Longer lists are cut into chunks, a workgroup each, which
// finds its share of the sorted list from a bit for every position; the chunks' sums
// are joined in order.
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
  uint32_t* cursor;                        // room taken, long lists, chunks
  uint4* chunks;                           // token, first of its chunks, chunk, chunks of the token
  float* sums;                             // [chunks][K]
  int chunk, most_chunks;
};

__device__ __forceinline__ int64_t token_at(const EmbedParams& p, int64_t m) {
  return p.wide ? static_cast<const int64_t*>(p.tokens)[m] : static_cast<const int32_t*>(p.tokens)[m];
}

// VW words of 4 bytes a lane, or one element where rows are not aligned to that (VW 0).
template <typename T, int VW>
struct Row {
  static constexpr int kElems = VW ? VW * 4 / (int)sizeof(T) : 1;
  static __device__ __forceinline__ void load(const T* src, float (&x)[kElems]) {
    if constexpr (VW == 0) {
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
    if constexpr (VW == 0) {
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
template <typename T, int VW>
__global__ __launch_bounds__(256) void embed_fwd_kernel(EmbedParams p) {
  typedef Row<T, VW> R;
  const int lane = threadIdx.x & 63;
  const int64_t m = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (m >= p.M) return;
  const int64_t v = token_at(p, m);
  T* out = static_cast<T*>(p.out) + m * p.so;
  const T* w = static_cast<const T*>(p.w) + (v >= 0 && v < p.V ? v : 0) * p.K;
  for (int k = lane * R::kElems; k < p.K; k += 64 * R::kElems) {
    float x[R::kElems];
    if (v >= 0 && v < p.V) {
      R::load(w + k, x);
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

__global__ __launch_bounds__(256) void embed_count_kernel(EmbedParams p) {
  const int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (m >= p.M) return;
  const int64_t v = token_at(p, m);
  if (v >= 0 && v < p.V) p.place[m] = atomicAdd(p.count + v, 1u);
}

// Room for each token's list, in no particular order, and the chunks of the long ones.
__global__ __launch_bounds__(256) void embed_room_kernel(EmbedParams p) {
  const int v = blockIdx.x * 256 + threadIdx.x, lane = threadIdx.x & 63;
  const uint32_t n = v < p.V ? p.count[v] : 0;
  uint32_t upto = n;  // room of the wave's lanes up to this one
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t o = __shfl_up(upto, d);
    if (lane >= d) upto += o;
  }
  uint32_t base = 0;
  if (lane == 63 && upto) base = atomicAdd(p.cursor, upto);
  base = __shfl(base, 63);
  if (n) p.start[v] = base + upto - n;
  if (n > 64) {
    const uint32_t parts = (n + p.chunk - 1) / p.chunk, first = atomicAdd(p.cursor + 1, parts);
    for (uint32_t c = 0; c < parts && first + c < (uint32_t)p.most_chunks; ++c) p.chunks[first + c] = uint4{(uint32_t)v, first, c, parts};
  }
}

__global__ __launch_bounds__(256) void embed_place_kernel(EmbedParams p) {
  const int64_t m = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (m >= p.M) return;
  const int64_t v = token_at(p, m);
  if (v >= 0 && v < p.V) p.list[p.start[v] + p.place[m]] = (uint32_t)m;
}

// The rows rows[0 .. n) of dout, in that order, from column k on. Loads of four are in flight.
template <typename T, int VW>
__device__ __forceinline__ void sum_rows(const EmbedParams& p, const uint32_t* rows, int n, int k, float (&s)[Row<T, VW>::kElems]) {
  typedef Row<T, VW> R;
  const T* dout = static_cast<const T*>(p.dout) + k;
#pragma unroll
  for (int i = 0; i < R::kElems; ++i) s[i] = 0.0f;
  for (int j0 = 0; j0 < n; j0 += 4) {
    float x[4][R::kElems];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j0 + j < n) R::load(dout + (int64_t)rows[j0 + j] * p.so, x[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j0 + j < n)
#pragma unroll
        for (int i = 0; i < R::kElems; ++i) s[i] += x[j][i];
  }
}

// A wave a token whose list is short: sorts it and sums its rows.
template <typename T, int VW>
__global__ __launch_bounds__(256) void embed_sum_kernel(EmbedParams p) {
  typedef Row<T, VW> R;
  __shared__ uint32_t sorted[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, v = blockIdx.x * 4 + wave;
  const int n = v < p.V ? __builtin_amdgcn_readfirstlane((int)p.count[v]) : 0;
  if (n > 0 && n <= 64) {
    const uint32_t mine = lane < n ? p.list[p.start[v] + lane] : 0xffffffffu;
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += (uint32_t)__builtin_amdgcn_readlane((int)mine, j) < mine ? 1 : 0;
    if (lane < n) sorted[wave][rank] = mine;
  }
  __syncthreads();
  if (v >= p.V || n > 64) return;
  T* dw = static_cast<T*>(p.dw) + (int64_t)v * p.K;
  for (int k = lane * R::kElems; k < p.K; k += 64 * R::kElems) {
    float s[R::kElems];
    sum_rows<T, VW>(p, sorted[wave], n, k, s);
#pragma unroll
    for (int i = 0; i < R::kElems; ++i) s[i] *= p.scale;
    R::store(dw + k, s);
  }
}

// A workgroup a chunk of a long list: the positions of ranks chunk c to chunk (c + 1).
// Bits of kWindow positions at a time say which are in the list; the bits before one are its rank.
constexpr int kWindow = 1 << 17, kMostChunk = 2048;
template <typename T, int VW>
__global__ __launch_bounds__(256) void embed_chunk_kernel(EmbedParams p) {
  typedef Row<T, VW> R;
  __shared__ uint32_t bits[kWindow / 32];
  __shared__ uint32_t rows[kMostChunk];
  __shared__ uint32_t upto[256];
  if (blockIdx.x >= min(p.cursor[1], (uint32_t)p.most_chunks)) return;  // uniform
  const uint4 c = p.chunks[blockIdx.x];
  const uint32_t n = p.count[c.x], from = c.z * p.chunk, to = min(n, from + p.chunk);
  const uint32_t* list = p.list + p.start[c.x];
  uint32_t before = 0;  // positions of the list in the windows before
  for (int64_t base = 0; base < p.M && before < to; base += kWindow) {
    const int words = (int)min((int64_t)kWindow, p.M - base + 31) / 32;
    for (int i = threadIdx.x; i < words; i += 256) bits[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
      const int64_t at = (int64_t)list[i] - base;
      if (at >= 0 && at < kWindow) atomicOr(bits + at / 32, 1u << (at & 31));
    }
    __syncthreads();
    // each thread counts the bits of a run of words; then the runs before it
    const int per = (words + 255) / 256, w0 = threadIdx.x * per;
    uint32_t mine = 0;
    for (int i = w0; i < min(w0 + per, words); ++i) mine += __popc(bits[i]);
    upto[threadIdx.x] = mine;
    __syncthreads();
    for (int d = 1; d < 256; d *= 2) {
      const uint32_t o = (int)threadIdx.x >= d ? upto[threadIdx.x - d] : 0;
      __syncthreads();
      upto[threadIdx.x] += o;
      __syncthreads();
    }
    uint32_t rank = before + upto[threadIdx.x] - mine;
    if (rank < to && rank + mine > from) {
      for (int i = w0; i < min(w0 + per, words); ++i)
        for (uint32_t w = bits[i]; w; w &= w - 1, ++rank)
          if (rank >= from && rank < to) rows[rank - from] = (uint32_t)(base + 32 * i + __ffs(w) - 1);
    }
    before += upto[255];
    __syncthreads();
  }
  const int count = (int)(to - from);
  for (int k = threadIdx.x * R::kElems; k < p.K; k += 256 * R::kElems) {
    float s[R::kElems];
    sum_rows<T, VW>(p, rows, count, k, s);
#pragma unroll
    for (int i = 0; i < R::kElems; ++i) p.sums[(int64_t)blockIdx.x * p.K + k + i] = s[i];
  }
}

// The chunks of a long list in order: a workgroup a chunk, of which the first of each list works.
template <typename T>
__global__ __launch_bounds__(256) void embed_join_kernel(EmbedParams p) {
  if (blockIdx.x >= min(p.cursor[1], (uint32_t)p.most_chunks)) return;
  const uint4 c = p.chunks[blockIdx.x];
  if (c.z != 0) return;
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
  // a list of n > 64 has n / chunk rounded up
  r.most_chunks = (int)(M / r.chunk + std::min<int64_t>(V, M / 65) + 1);
  r.clear = 64 + V;  // cursors on a line of their own, counts
  r.start = align256(r.clear * 4);
  r.place = r.start + align256(V * 4);
  r.list = r.place + align256(M * 4);
  r.chunks = r.list + align256(M * 4);
  r.sums = r.chunks + align256((int64_t)r.most_chunks * 16);
  r.total = r.sums + align256((int64_t)r.most_chunks * K * 4);
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
  auto fn = size == 4 ? (vec ? embed_fwd_kernel<float, 4> : embed_fwd_kernel<float, 0>)
                      : (vec ? embed_fwd_kernel<__bf16, 4> : embed_fwd_kernel<__bf16, 0>);
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
  const dim3 rows((unsigned)((a->M + 255) / 256)), words((unsigned)((a->V + 255) / 256));
  hipLaunchKernelGGL(embed_clear_kernel, dim3((unsigned)((plan.clear + 255) / 256)), dim3(256), 0, stream, p.cursor, plan.clear);
  GS_CHECK_HIP(hipGetLastError());
  hipLaunchKernelGGL(embed_count_kernel, rows, dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  hipLaunchKernelGGL(embed_room_kernel, words, dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  hipLaunchKernelGGL(embed_place_kernel, rows, dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  const bool vec = aligned16(a->dw, a->K, size) && aligned16(a->dout, a->sdo, size);
  auto sum = size == 4 ? (vec ? embed_sum_kernel<float, 4> : embed_sum_kernel<float, 0>)
                       : (vec ? embed_sum_kernel<__bf16, 4> : embed_sum_kernel<__bf16, 0>);
  hipLaunchKernelGGL(sum, dim3((unsigned)((a->V + 3) / 4)), dim3(256), 0, stream, p);
  GS_CHECK_HIP(hipGetLastError());
  if (a->M > 64) {
    auto chunk = size == 4 ? (vec ? embed_chunk_kernel<float, 4> : embed_chunk_kernel<float, 0>)
                           : (vec ? embed_chunk_kernel<__bf16, 4> : embed_chunk_kernel<__bf16, 0>);
    hipLaunchKernelGGL(chunk, dim3((unsigned)plan.most_chunks), dim3(256), 0, stream, p);
    GS_CHECK_HIP(hipGetLastError());
    hipLaunchKernelGGL(size == 4 ? embed_join_kernel<float> : embed_join_kernel<__bf16>, dim3((unsigned)plan.most_chunks, 4),
                       dim3(256), 0, stream, p);
    GS_CHECK_HIP(hipGetLastError());
  }
  return GS_OK;
}
