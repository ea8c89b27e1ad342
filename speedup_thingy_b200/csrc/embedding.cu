// Embedding lookup with a scale, and the table's gradient by sorted tokens (operator table: k_embedding).
//
//   y_t = scale * w[id_t],     dw_v = scale * sum over { t : id_t = v } of dy_t,  in fp32, rounded once
//
// The gradient's addends meet in the order of the tokens, whatever the launch: the token positions are sorted by (id, position), a
// thread adds its columns of RANGE consecutive sorted rows, what a range adds for an id that reaches beyond it goes to a partial, and
// the range in which such an id begins adds the partials in order.  No atomics; rows that no token names are zeros.
//
// The sort counts: the place of token i in its chunk of CHUNK tokens is the number of tokens j of the chunk with
// (id_j, j) < (id_i, i); a second launch adds, for every other chunk, how many of its ids come before, by binary search.

#include <cuda_fp16.h>

#include "rte_common.cuh"

namespace {

constexpr int EO_CHUNK = 4096, EO_RANGE = 32, EO_LANES = 8;          // tokens a chunk, sorted rows a range, threads that count for one token

// `BYTES` of a row at a time, as fp32
template <typename T, int BYTES> struct Piece {
  static constexpr int N = BYTES / (int)sizeof(T);
  float v[N];
};
template <typename T> __device__ __forceinline__ float as_float(T v) { return (float)v; }
template <typename T, int BYTES> struct Raw;
template <typename T> struct Raw<T, 16> { using type = uint4; };
template <typename T> struct Raw<T, 8> { using type = uint2; };
template <typename T> struct Raw<T, 4> { using type = uint32_t; };
template <typename T> struct Raw<T, 2> { using type = uint16_t; };

template <typename T, int BYTES>
__device__ __forceinline__ Piece<T, BYTES> unpack(typename Raw<T, BYTES>::type raw) {
  T t[BYTES / sizeof(T)];
  memcpy(t, &raw, BYTES);
  Piece<T, BYTES> p;
#pragma unroll
  for (int i = 0; i < p.N; ++i) p.v[i] = as_float(t[i]);
  return p;
}
template <typename T, int BYTES>
__device__ __forceinline__ typename Raw<T, BYTES>::type pack(const Piece<T, BYTES>& p, float scale) {
  T t[BYTES / sizeof(T)];
#pragma unroll
  for (int i = 0; i < p.N; ++i) t[i] = (T)(p.v[i] * scale);
  typename Raw<T, BYTES>::type raw;
  memcpy(&raw, t, BYTES);
  return raw;
}

// A thread per piece of a row.
template <typename T, int BYTES>
__global__ void __launch_bounds__(256)
embedding_fwd_kernel(const int64_t* __restrict__ ids, long long n, const T* __restrict__ table, int V, int pieces, float scale, T* __restrict__ out, int* status) {
  rte::after_previous_grid();
  using R = typename Raw<T, BYTES>::type;
  const R* w = reinterpret_cast<const R*>(table);
  R* y = reinterpret_cast<R*>(out);
  const long long total = n * pieces;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const long long t = i / pieces, id = ids[t];
    const int c = int(i - t * pieces);
    if (id < 0 || id >= V) {
      if (status && c == 0) atomicExch(status, RTE_DEV_INDEX_OUT_OF_RANGE);
      y[i] = R{};
    } else {
      y[i] = pack<T, BYTES>(unpack<T, BYTES>(w[id * pieces + c]), scale);
    }
  }
}

struct EoScratch {
  int *chunk_id, *chunk_tok;      // [n]: every chunk sorted
  int *id, *tok;                  // [n]: all sorted (the same two where there is one chunk)
  float* part;                    // [ranges][2][d]: what a range adds for an id that began before it | that goes on after it
};
inline size_t eo_layout(char* at, long long n, int d, EoScratch* s) {
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t list = up((size_t)n * 4), lists = n > EO_CHUNK ? 4 : 2, part = up((size_t)rte::ceil_div64(n, EO_RANGE) * 2 * d * 4);
  if (s) {
    s->chunk_id = reinterpret_cast<int*>(at);
    s->chunk_tok = reinterpret_cast<int*>(at + list);
    s->id = reinterpret_cast<int*>(at + (lists - 2) * list);
    s->tok = reinterpret_cast<int*>(at + (lists - 1) * list);
    s->part = reinterpret_cast<float*>(at + lists * list);
  }
  return lists * list + part;
}

// Ids that take no gradient (padding, out of range) count as V: behind all others.
__device__ __forceinline__ int eo_id(long long v, int V, long long padding, int* status) {
  if (v >= 0 && v < V) return v == padding ? V : (int)v;
  if (status) atomicExch(status, RTE_DEV_INDEX_OUT_OF_RANGE);
  return V;
}

// blockIdx.y: chunk; a CTA places 256 / EO_LANES of its tokens, EO_LANES threads counting for each.
__global__ void __launch_bounds__(256)
embedding_rank_kernel(const int64_t* __restrict__ ids, int n, int V, long long padding, EoScratch S, int* status) {
  rte::after_previous_grid();
  __shared__ __align__(16) int id[EO_CHUNK];
  const int first = blockIdx.y * EO_CHUNK, count = min(EO_CHUNK, n - first), tid = threadIdx.x;
  if ((int)blockIdx.x * (256 / EO_LANES) >= count) return;
  for (int j = tid; j < EO_CHUNK; j += 256) id[j] = j < count ? eo_id(ids[first + j], V, padding, status) : 0x7fffffff;
  __syncthreads();
  const int i = blockIdx.x * (256 / EO_LANES) + tid / EO_LANES, sub = tid % EO_LANES;
  const int mine = i < count ? id[i] : 0;
  int rank = 0;
  for (int q = sub; q < (count + 3) / 4; q += EO_LANES) {
    const int4 v = reinterpret_cast<const int4*>(id)[q];
    const int e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) rank += e[u] < mine + (4 * q + u < i);
  }
#pragma unroll
  for (int o = EO_LANES / 2; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
  if (sub == 0 && i < count) {
    S.chunk_id[first + rank] = mine;
    S.chunk_tok[first + rank] = first + i;
  }
}

// how many of the `count` sorted ids are below `limit`
__device__ __forceinline__ int below(const int* __restrict__ ids, int count, long long limit) {
  int lo = 0, hi = count;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ids[mid] < limit) lo = mid + 1; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(256)
embedding_merge_kernel(EoScratch S, int n) {
  rte::after_previous_grid();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int chunk = i / EO_CHUNK, id = S.chunk_id[i];
  int at = i - chunk * EO_CHUNK;
  for (int c = 0; c * EO_CHUNK < n; ++c)
    if (c != chunk) at += below(S.chunk_id + c * EO_CHUNK, min(EO_CHUNK, n - c * EO_CHUNK), (long long)id + (c < chunk));
  S.id[at] = id;
  S.tok[at] = S.chunk_tok[i];
}

// blockIdx.x < ranges: a range's sums, its pieces of columns dealt to blockIdx.y; beyond: zeros of 128 table rows that no token names.
template <typename T, int BYTES>
__global__ void __launch_bounds__(128)
embedding_sum_kernel(const T* __restrict__ dy, EoScratch S, int n, int V, int pieces, int d, float scale, T* __restrict__ dtable, int ranges) {
  rte::after_previous_grid();
  using R = typename Raw<T, BYTES>::type;
  using P = Piece<T, BYTES>;
  R* out = reinterpret_cast<R*>(dtable);
  const int tid = threadIdx.x;
  if ((int)blockIdx.x >= ranges) {
    __shared__ int named[128];
    const long long v0 = 128LL * (blockIdx.x - ranges);
    const int v = (int)min(v0 + tid, (long long)V);
    const int at = below(S.id, n, v);
    named[tid] = at < n && S.id[at] == v;
    __syncthreads();
    for (int r = 0; r < 128 && v0 + r < V; ++r)
      if (!named[r])
        for (int c = blockIdx.y * 128 + tid; c < pieces; c += gridDim.y * 128) out[(v0 + r) * pieces + c] = R{};
    return;
  }
  __shared__ int id[EO_RANGE + 2], tok[EO_RANGE];
  const int a = blockIdx.x * EO_RANGE, count = min(EO_RANGE, n - a);
  for (int i = tid; i < count + 2; i += 128) {
    const int at = a - 1 + i;
    id[i] = at >= 0 && at < n ? S.id[at] : -1;
  }
  for (int i = tid; i < count; i += 128) tok[i] = S.tok[a + i];
  __syncthreads();
  const R* g = reinterpret_cast<const R*>(dy);
  for (int c = blockIdx.y * 128 + tid; c < pieces; c += gridDim.y * 128) {
    P acc;
    int begin = 0;
    for (int i = 0; i < count && id[i + 1] < V; ++i) {
      const P x = unpack<T, BYTES>(g[(long long)tok[i] * pieces + c]);
      if (i == begin) acc = x;
      else
#pragma unroll
        for (int u = 0; u < P::N; ++u) acc.v[u] += x.v[u];
      if (i + 1 < count && id[i + 2] == id[i + 1]) continue;
      const bool before = begin == 0 && id[0] == id[1], after = i + 1 == count && id[i + 2] == id[i + 1];
      if (before || after) {
        float* p = S.part + ((size_t)blockIdx.x * 2 + !before) * d + c * P::N;
#pragma unroll
        for (int u = 0; u < P::N; ++u) p[u] = acc.v[u];
      } else {
        out[(long long)id[i + 1] * pieces + c] = pack<T, BYTES>(acc, scale);
      }
      begin = i + 1;
    }
  }
}

// The range in which an id begins that reaches beyond it adds what the ranges behind it have of it, in their order.
template <typename T>
__global__ void __launch_bounds__(128)
embedding_join_kernel(EoScratch S, int n, int V, int d, float scale, T* __restrict__ dtable) {
  rte::after_previous_grid();
  const int a = blockIdx.x * EO_RANGE, end = a + EO_RANGE;
  if (end >= n) return;
  const int v = S.id[end];
  if (v >= V || S.id[end - 1] != v || (S.id[a] == v && a > 0 && S.id[a - 1] == v)) return;
  const int last = (below(S.id, n, (long long)v + 1) - 1) / EO_RANGE;
  for (int c = blockIdx.y * 128 + threadIdx.x; c < d; c += gridDim.y * 128) {
    float s = S.part[((size_t)blockIdx.x * 2 + 1) * d + c];
    for (int r = blockIdx.x + 1; r <= last; ++r) s += S.part[(size_t)r * 2 * d + c];
    dtable[(long long)v * d + c] = (T)(s * scale);
  }
}

bool type_ok(int type) { return type == RTE_TYPE_BF16 || type == RTE_TYPE_F16 || type == RTE_TYPE_F32; }
// the widest pieces that every row of the two tensors starts on
int piece_bytes(const void* a, const void* b, long long row_bytes) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | (uintptr_t)row_bytes;
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

template <typename T, int BYTES>
void launch_fwd(const int64_t* ids, long long n, const void* table, int V, int d, float scale, void* out, int* status, cudaStream_t st) {
  const int pieces = d * (int)sizeof(T) / BYTES;
  const long long ctas = rte::ceil_div64(n * pieces, 256);
  rte::launch(embedding_fwd_kernel<T, BYTES>, (unsigned)(ctas < 148 * 64 ? ctas : 148 * 64), 256, 0, st, ids, n, static_cast<const T*>(table), V, pieces, scale,
              static_cast<T*>(out), status);
}
template <typename T, int BYTES>
void launch_sum(const void* dy, const EoScratch& s, int n, int V, int d, float scale, void* dtable, cudaStream_t st) {
  const int pieces = d * (int)sizeof(T) / BYTES, ranges = rte::ceil_div(n, EO_RANGE);
  const dim3 grid(ranges + rte::ceil_div(V, 128), (unsigned)min(rte::ceil_div(pieces, 128), 64));
  rte::launch(embedding_sum_kernel<T, BYTES>, grid, 128, 0, st, static_cast<const T*>(dy), s, n, V, pieces, d, scale, static_cast<T*>(dtable), ranges);
  if (n > EO_RANGE)
    rte::launch(embedding_join_kernel<T>, dim3(ranges - 1, (unsigned)min(rte::ceil_div(d, 128), 64)), 128, 0, st, s, n, V, d, scale, static_cast<T*>(dtable));
}

}  // namespace

#define ST(s) static_cast<cudaStream_t>(s)
#define BY_PIECE(type, bytes, CALL)                                   \
  do {                                                                \
    if (type == RTE_TYPE_F32) {                                       \
      if (bytes == 16) CALL(float, 16);                               \
      else if (bytes == 8) CALL(float, 8);                            \
      else CALL(float, 4);                                            \
    } else if (type == RTE_TYPE_BF16) {                               \
      if (bytes == 16) CALL(__nv_bfloat16, 16);                       \
      else if (bytes == 8) CALL(__nv_bfloat16, 8);                    \
      else if (bytes == 4) CALL(__nv_bfloat16, 4);                    \
      else CALL(__nv_bfloat16, 2);                                    \
    } else {                                                          \
      if (bytes == 16) CALL(__half, 16);                              \
      else if (bytes == 8) CALL(__half, 8);                           \
      else if (bytes == 4) CALL(__half, 4);                           \
      else CALL(__half, 2);                                           \
    }                                                                 \
  } while (0)

extern "C" int rte_embedding_fwd(const int64_t* ids, int64_t n, const void* table, int32_t type, int32_t V, int32_t d, float scale, void* out, int32_t* status,
                                 rte_stream_t stream) {
  RTE_CHECK_ARG(ids && table && out && type_ok(type) && n > 0 && V > 0 && d > 0);
  const int bytes = piece_bytes(table, out, (long long)d * (type == RTE_TYPE_F32 ? 4 : 2));
  if (type == RTE_TYPE_F32 && bytes < 4) return RTE_ERR_ALIGNMENT;
#define CALL(T, B) launch_fwd<T, B>(ids, n, table, V, d, scale, out, status, ST(stream))
  BY_PIECE(type, bytes, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}

extern "C" int64_t rte_embedding_bwd_scratch(int64_t n, int32_t d) {
  if (n <= 0 || d <= 0 || n > RTE_EMBEDDING_MAX_TOKENS) return 0;
  return (int64_t)eo_layout(nullptr, n, d, nullptr);
}

extern "C" int rte_embedding_bwd(const int64_t* ids, int64_t n, const void* dy, int32_t type, int32_t V, int32_t d, float scale, int64_t padding_idx, void* dtable,
                                 void* scratch, int64_t scratch_bytes, int32_t* status, rte_stream_t stream) {
  RTE_CHECK_ARG(ids && dy && dtable && scratch && type_ok(type) && n > 0 && n <= RTE_EMBEDDING_MAX_TOKENS && V > 0 && V < 0x7fffffff && d > 0);
  if (scratch_bytes < rte_embedding_bwd_scratch(n, d)) return RTE_ERR_SCRATCH_CAPACITY;
  if (reinterpret_cast<uintptr_t>(scratch) & 15) return RTE_ERR_ALIGNMENT;
  const int bytes = piece_bytes(dy, dtable, (long long)d * (type == RTE_TYPE_F32 ? 4 : 2));
  if (type == RTE_TYPE_F32 && bytes < 4) return RTE_ERR_ALIGNMENT;
  EoScratch s;
  eo_layout(static_cast<char*>(scratch), n, d, &s);
  const int chunks = (int)rte::ceil_div64(n, EO_CHUNK), in_chunk = (int)(n < EO_CHUNK ? n : EO_CHUNK);
  rte::launch(embedding_rank_kernel, dim3(rte::ceil_div(in_chunk, 256 / EO_LANES), chunks), 256, 0, ST(stream), ids, (int)n, V, padding_idx, s, status);
  if (chunks > 1) rte::launch(embedding_merge_kernel, (unsigned)rte::ceil_div64(n, 256), 256, 0, ST(stream), s, (int)n);
#define CALL(T, B) launch_sum<T, B>(dy, s, (int)n, V, d, scale, dtable, ST(stream))
  BY_PIECE(type, bytes, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}
