// Embedding lookup with a scale, and the table's gradient by sorted tokens (operator table: k_embedding).
//
//   y_t = scale * w[id_t],     dw_v = scale * sum over { t : id_t = v } of dy_t,  in fp32, rounded once
//
// The gradient's addends meet in the order of the tokens, whatever the launch: the token positions are sorted by (id, position), a
// thread adds its columns of a range of consecutive sorted rows, what a range adds for an id that reaches beyond it goes to a
// partial, and those of one id are added in order; an id that ends within the next range is finished by the one in which it
// begins.  No atomics on values; rows that no token names are zeros.
//
// The sort takes a pass per digit of the id, each stable: a token's place is the number of tokens with a smaller digit, those with its own
// in CTAs before, in warps before, and in its warp before it.  Up to SORT_ONE tokens are one cluster's, which exchanges its CTAs' counts
// (digits of up to 8 bits, all passes in one launch).  More are counted by CTAs, and a pass leaves the next digit's counts behind, so that a sort of two digits (of up to 10 bits: tables
// of up to 2^20 rows) is three launches.  A few tokens' gradient is one launch: the cluster that sorts them adds their rows too.

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "rte_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int SORT_ONE = 49152, ONE_CTAS = 8, ONE_BITS = 8;          // tokens that one cluster sorts, its CTAs, the bits of its digits
constexpr int SORT_THREADS = 256, SORT_CTAS = 296;                   // of a sort's launch; CTAs at most
constexpr int SORT_BITS = 10;                                        // of a digit, at most
constexpr int ROWS_AHEAD = 8, MAX_RANGE = 64;                        // rows a thread has in flight; sorted rows of a range at most

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

// 128 threads as groups of `tpr`, a power of two, a thread per piece of a row and further ones where a row has more than 128.
int threads_per_row(int pieces) {
  int t = 1;
  while (t < pieces && t < 128) t *= 2;
  return t;
}

// A group takes TOKENS_AHEAD tokens at a time: a thread has that many rows in flight and no division per piece (one piece a thread and a
// division: 8192 x 1024 bf16 7.0 -> 5.1 us, 33333 x 770 fp32 41 -> 29.5, 131072 x 2048 bf16 123 -> 106 = 5 TB/s of writes).
constexpr int TOKENS_AHEAD = 4;
template <typename T, int BYTES>
__global__ void __launch_bounds__(128)
embedding_fwd_kernel(const int64_t* __restrict__ ids, long long n, const T* __restrict__ table, int V, int pieces, int tpr, float scale, T* __restrict__ out, int* status) {
  rte::after_previous_grid();
  using R = typename Raw<T, BYTES>::type;
  const R* w = reinterpret_cast<const R*>(table);
  R* y = reinterpret_cast<R*>(out);
  const int lane = threadIdx.x % tpr, groups = 128 / tpr;
  for (long long t = ((long long)blockIdx.x * groups + threadIdx.x / tpr) * TOKENS_AHEAD; t < n; t += (long long)gridDim.x * groups * TOKENS_AHEAD) {
    long long id[TOKENS_AHEAD];
    float by[TOKENS_AHEAD];                                        // zero times zero without a row, whatever the scale
#pragma unroll
    for (int u = 0; u < TOKENS_AHEAD; ++u) {
      id[u] = t + u < n ? ids[t + u] : 0;
      if (id[u] < 0 || id[u] >= V) {
        if (status && lane == 0 && blockIdx.y == 0) atomicExch(status, RTE_DEV_INDEX_OUT_OF_RANGE);
        id[u] = -1;
      }
      by[u] = id[u] >= 0 ? scale : 0.f;
    }
    for (int c = blockIdx.y * tpr + lane; c < pieces; c += gridDim.y * tpr) {
      R r[TOKENS_AHEAD];
#pragma unroll
      for (int u = 0; u < TOKENS_AHEAD; ++u) r[u] = id[u] >= 0 ? w[id[u] * pieces + c] : R{};
#pragma unroll
      for (int u = 0; u < TOKENS_AHEAD; ++u)
        if (t + u < n) y[(t + u) * pieces + c] = pack<T, BYTES>(unpack<T, BYTES>(r[u]), by[u]);
    }
  }
}

// ---------------------------------------------------------------- the gradient's workspace
struct Digits { int passes, bits; };           // of ids 0 .. V (V: takes no gradient)
Digits digits_of(int V, int most) {
  int b = 1;
  while (b < 31 && V >> b) ++b;
  const int passes = (b + most - 1) / most;
  return {passes, (b + passes - 1) / passes};
}
struct EoScratch {
  int *id, *tok;                // [n]: sorted
  int *id2, *tok2;              // [n]: between passes
  int* hist;                    // [passes][sort CTAs][1 << bits]
  int2* joins;                  // (range, id): ranges in which an id begins that fills the next one too and goes on
  int* join_count;
  float* part;                  // [ranges][2][d]: what a range adds for an id that began before it | that goes on behind it
};
// Tokens that a thread of a sort CTA places at a time: few while the CTAs are few (all of them read all of their counts).
int sort_each(long long n) { return n <= 65536 ? 4 : 8; }
int sort_span(long long n) {                                          // tokens of a sort CTA
  const int tile = SORT_THREADS * sort_each(n);
  return (int)rte::ceil_div64(rte::ceil_div64(n, tile), SORT_CTAS) * tile;
}
int range_of(long long n) { return n >= 65536 ? MAX_RANGE : n >= 32768 ? 32 : n >= 8192 ? 16 : 8; }
size_t eo_layout(char* at, long long n, int d, EoScratch* s) {
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  const size_t list = up((size_t)n * 4), ranges = (size_t)rte::ceil_div64(n, range_of(n));
  // (three digits of 10 bits and one more pass: what a table of any size takes)
  const size_t hist = n > SORT_ONE ? up((size_t)4 * rte::ceil_div64(n, sort_span(n)) * (1 << SORT_BITS) * 4) : 0;
  const size_t lists = 4;
  if (s) {
    s->id = reinterpret_cast<int*>(at);
    s->tok = reinterpret_cast<int*>(at + list);
    s->id2 = reinterpret_cast<int*>(at + 2 * list);
    s->tok2 = reinterpret_cast<int*>(at + 3 * list);
    s->hist = reinterpret_cast<int*>(at + lists * list);
    s->join_count = reinterpret_cast<int*>(at + lists * list + hist);
    s->joins = reinterpret_cast<int2*>(s->join_count + 64);
    s->part = reinterpret_cast<float*>(at + lists * list + hist + 256 + up(ranges * 8));
  }
  return lists * list + hist + 256 + up(ranges * 8) + up(ranges * 2 * d * 4);
}

// Ids that take no gradient (padding, out of range) count as V: behind all others.
__device__ __forceinline__ int eo_id(long long v, int V, long long padding, int* status) {
  if (v >= 0 && v < V) return v == padding ? V : (int)v;
  if (status) atomicExch(status, RTE_DEV_INDEX_OUT_OF_RANGE);
  return V;
}

// Zeros, by the CTAs that a sort's launch has beside those that sort: a sort leaves most of the memory's time to them.
struct Fill { char* at; long long bytes; };
__device__ __forceinline__ void fill(const Fill& f, int cta, int ctas) {
  const int tid = threadIdx.x, nt = blockDim.x;
  const long long head = min(f.bytes, (long long)(-reinterpret_cast<uintptr_t>(f.at) & 15)), body = (f.bytes - head) / 16;
  uint4* q = reinterpret_cast<uint4*>(f.at + head);
  for (long long i = (long long)cta * nt + tid; i < body; i += (long long)ctas * nt) q[i] = make_uint4(0, 0, 0, 0);
  if (cta == 0) {
    for (long long i = tid; i < head; i += nt) f.at[i] = 0;
    for (long long i = head + body * 16 + tid; i < f.bytes; i += nt) f.at[i] = 0;
  }
}

// ---------------------------------------------------------------- sort
// The lanes with this lane's digit (of `bits` bits), those that bring none apart: a vote per bit.
__device__ __forceinline__ uint32_t same_digit(int digit, bool brings, int bits) {
  uint32_t same = __ballot_sync(0xffffffffu, brings);
  if (!brings) same = ~same;
#pragma unroll
  for (int b = 0; b < SORT_BITS; ++b) {
    if (b >= bits) break;
    const bool one = digit >> b & 1;
    const uint32_t ones = __ballot_sync(0xffffffffu, one);
    same &= one ? ones : ~ones;
  }
  return same;
}
// Exclusive sums over the block's threads.
__device__ __forceinline__ int sums_before(int v, int* warp_total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int upto = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int u = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += u; }
  if (lane == 31) warp_total[warp] = upto;
  __syncthreads();
  int at = upto - v;
  for (int w = 0; w < warp; ++w) at += warp_total[w];
  return at;
}

// Up to SORT_ONE tokens by the first cluster, a run of neighbouring tokens per CTA, up to 24 of them a thread; the other clusters fill.  One
// CTA of 1024 threads took 21 us for 8192 tokens, most of it the rounds of votes on one SM.  Whole gradients, us, launches per digit | one
// cluster: 16384 x 1024 bf16 of 32768 45 | 37.6, 30000 x 1024 67 | 55, 30000 x 256 of 2000 49 | 38, 45000 x 1024 of 131072 104 | 96.
// EACH: tokens of a thread at most.  Ends with a cluster's barrier.
template <int EACH>
__device__ __forceinline__ void sort_one(const int64_t* __restrict__ ids, int n, int V, long long padding, const EoScratch& S, int passes, int bits, int* status) {
  constexpr int WARPS = SORT_THREADS / 32, BINS = 1 << ONE_BITS;
  static_assert(BINS == SORT_THREADS, "a thread per digit");
  __shared__ int base[BINS], count[BINS], warp_total[WARPS];
  __shared__ unsigned short in_warp[WARPS][BINS];
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank_in = (int)cluster.block_rank();
  const int each = (n + ONE_CTAS * SORT_THREADS - 1) / (ONE_CTAS * SORT_THREADS);      // rounds of a warp
  const int first = (rank_in * WARPS + warp) * 32 * each + lane;     // a warp's tokens are neighbours
  if (blockIdx.x == 0 && tid == 0) *S.join_count = 0;
  int id[EACH], tok[EACH], rank[EACH];
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    const bool to_first = (passes - 1 - pass) % 2 == 0;
    int *id_out = to_first ? S.id : S.id2, *tok_out = to_first ? S.tok : S.tok2;
    const int *id_in = to_first ? S.id2 : S.id, *tok_in = to_first ? S.tok2 : S.tok;
    if (pass == 0) {
      int64_t v[EACH];                                               // (all requested before the first is looked at)
#pragma unroll
      for (int e = 0; e < EACH; ++e) v[e] = e < each && first + 32 * e < n ? ids[first + 32 * e] : 0;
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const bool in = e < each && first + 32 * e < n;
        id[e] = in ? eo_id(v[e], V, padding, status) : -1;
        tok[e] = first + 32 * e;
      }
    } else {
#pragma unroll
      for (int e = 0; e < EACH; ++e) {
        const bool in = e < each && first + 32 * e < n;
        id[e] = in ? __ldcg(id_in + first + 32 * e) : -1;
        tok[e] = in ? __ldcg(tok_in + first + 32 * e) : 0;
      }
    }
#pragma unroll
    for (int w = 0; w < WARPS; ++w) in_warp[w][tid] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      if (e >= each) break;
      const int digit = id[e] >> shift & (BINS - 1) & ((1 << bits) - 1);
      const uint32_t same = same_digit(digit, id[e] >= 0, bits);
      rank[e] = in_warp[warp][digit] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (id[e] >= 0 && same >> lane == 1) in_warp[warp][digit] += __popc(same);               // (the last of them)
      __syncwarp();
    }
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) { const int v = in_warp[w][tid]; in_warp[w][tid] = (unsigned short)sum; sum += v; }
    count[tid] = sum;
    cluster.sync();
    int total = 0, before = 0;
#pragma unroll
    for (int c = 0; c < ONE_CTAS; ++c) {
      const int v = cluster.map_shared_rank(count, c)[tid];
      total += v;
      before += c < rank_in ? v : 0;
    }
    base[tid] = sums_before(total, warp_total) + before;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      if (id[e] < 0) continue;
      const int digit = id[e] >> shift & ((1 << bits) - 1), at = base[digit] + in_warp[warp][digit] + rank[e];
      id_out[at] = id[e];
      tok_out[at] = tok[e];
    }
    cluster.sync();                                                  // (every CTA's places are written, its counts read)
  }
}
__global__ void __cluster_dims__(ONE_CTAS, 1, 1) __launch_bounds__(SORT_THREADS)
embedding_sort_kernel(const int64_t* __restrict__ ids, int n, int V, long long padding, EoScratch S, int passes, int bits, Fill f, int* status) {
  rte::after_previous_grid();
  if (blockIdx.x >= ONE_CTAS) return fill(f, blockIdx.x - ONE_CTAS, gridDim.x - ONE_CTAS);
  sort_one<SORT_ONE / ONE_CTAS / SORT_THREADS>(ids, n, V, padding, S, passes, bits, status);
}

// The first digit's counts of every sort CTA's tokens; the other passes' counts are cleared.
__global__ void __launch_bounds__(SORT_THREADS)
embedding_count_kernel(const int64_t* __restrict__ ids, int n, int V, long long padding, EoScratch S, int passes, int bits, int span, int ctas, Fill f, int* status) {
  rte::after_previous_grid();
  if ((int)blockIdx.x >= ctas) return fill(f, blockIdx.x - ctas, gridDim.x - ctas);
  __shared__ int count[1 << SORT_BITS];
  const int tid = threadIdx.x, bins = 1 << bits;
  for (int b = tid; b < bins; b += SORT_THREADS) count[b] = 0;
  if (blockIdx.x == 0 && tid == 0) *S.join_count = 0;
  __syncthreads();
  const int begin = blockIdx.x * span, end = min(begin + span, n);
  for (int i0 = begin + tid; i0 < end; i0 += 8 * SORT_THREADS) {
    int64_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = i0 + e * SORT_THREADS < end ? ids[i0 + e * SORT_THREADS] : 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i0 + e * SORT_THREADS < end) atomicAdd(&count[eo_id(v[e], V, padding, status) & (bins - 1)], 1);
  }
  __syncthreads();
  for (int b = tid; b < bins; b += SORT_THREADS) {
    S.hist[blockIdx.x * bins + b] = count[b];
    for (int p = 1; p < passes; ++p) S.hist[(p * ctas + blockIdx.x) * bins + b] = 0;
  }
}

// One pass: the tokens of a CTA, EACH per thread at a time, go to their places by digit `pass`.
template <int EACH>
__global__ void __launch_bounds__(SORT_THREADS)
embedding_place_kernel(const int64_t* __restrict__ ids, const int* __restrict__ id_in, const int* __restrict__ tok_in, int* __restrict__ id_out, int* __restrict__ tok_out,
                       int* __restrict__ hist, int n, int V, long long padding, int pass, int passes, int bits, int span, int ctas, Fill f) {
  rte::after_previous_grid();
  if ((int)blockIdx.x >= ctas) return fill(f, blockIdx.x - ctas, gridDim.x - ctas);
  constexpr int WARPS = SORT_THREADS / 32, TILE = SORT_THREADS * EACH, BINS_EACH = (1 << SORT_BITS) / SORT_THREADS;
  __shared__ int base[1 << SORT_BITS];                             // where the next token of a digit goes
  __shared__ unsigned short in_warp[WARPS][1 << SORT_BITS];
  __shared__ int warp_total[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = 1 << bits, shift = pass * bits;
  {                                                              // a thread has BINS_EACH neighbouring digits
    const int* h = hist + (size_t)pass * ctas * bins;
    int total[BINS_EACH] = {}, before[BINS_EACH] = {};
    const int each = (bins + SORT_THREADS - 1) / SORT_THREADS;
    for (int u = 0; u < each; ++u) {
      const int b = tid * each + u;
      if (b >= bins) break;
#pragma unroll 16
      for (int c = 0; c < ctas; ++c) {
        const int v = h[c * bins + b];
        total[u] += v;
        before[u] += c < (int)blockIdx.x ? v : 0;
      }
    }
    int sum = 0;
#pragma unroll
    for (int u = 0; u < BINS_EACH; ++u) sum += total[u];
    int at = sums_before(sum, warp_total);
    for (int u = 0; u < each; ++u) {
      const int b = tid * each + u;
      if (b < bins) base[b] = at + before[u];
      at += total[u];
    }
  }
  const int end = min((int)blockIdx.x * span + span, n);
  for (int tile = blockIdx.x * span; tile < end; tile += TILE) {
    for (int b = tid; b < WARPS * bins; b += SORT_THREADS) in_warp[b >> bits][b & (bins - 1)] = 0;
    __syncthreads();
    int id[EACH], tok[EACH], rank[EACH];
    const int first = tile + warp * 32 * EACH + lane;              // a warp's tokens are neighbours
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int i = first + 32 * e;
      id[e] = i < end ? (pass == 0 ? eo_id(ids[i], V, padding, nullptr) : id_in[i]) : -1;
      tok[e] = i < end ? (pass == 0 ? i : tok_in[i]) : 0;
    }
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const int digit = id[e] >> shift & (bins - 1);
      const uint32_t same = same_digit(digit, id[e] >= 0, bits);
      rank[e] = in_warp[warp][digit] + __popc(same & ((1u << lane) - 1));
      __syncwarp();
      if (id[e] >= 0 && same >> lane == 1) in_warp[warp][digit] += __popc(same);           // (the last of them)
      __syncwarp();
    }
    __syncthreads();
    int in_tile[BINS_EACH] = {};
#pragma unroll
    for (int u = 0; u < BINS_EACH; ++u) {                          // every warp's counts become where its first token goes, within the tile
      const int b = tid + u * SORT_THREADS;
      if (b >= bins) break;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) { const int v = in_warp[w][b]; in_warp[w][b] = (unsigned short)in_tile[u]; in_tile[u] += v; }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      if (id[e] < 0) continue;
      const int digit = id[e] >> shift & (bins - 1), at = base[digit] + in_warp[warp][digit] + rank[e];
      id_out[at] = id[e];
      tok_out[at] = tok[e];
      if (pass + 1 < passes) atomicAdd(&hist[((size_t)(pass + 1) * ctas + at / span) * bins + (id[e] >> (shift + bits) & (bins - 1))], 1);
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < BINS_EACH; ++u)
      if (tid + u * SORT_THREADS < bins) base[tid + u * SORT_THREADS] += in_tile[u];
  }
}

// ---------------------------------------------------------------- sums
// how many of the `count` sorted ids are below `limit`
__device__ __forceinline__ int below(const int* __restrict__ ids, int count, long long limit) {
  int lo = 0, hi = count;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ids[mid] < limit) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// Bound by HBM for long batches (131072 x 2048 bf16: 115 us for 537 MB read and 100 MB written), by the latency of a few rounds of
// loads for short ones (8192 x 1024: about 9 us).
// Groups of tpr threads: one adds the rows of a range, a piece of the columns per thread.  CTAs behind `range_ctas`: zeros of ZERO_ROWS table
// rows that no token names, where the sort's launches have not filled the table.
constexpr int ZERO_ROWS = 64, MIN_TPR = 8;
template <int RANGE> struct Sorted { int ids[128 / MIN_TPR][2 * RANGE + 2], toks[128 / MIN_TPR][2 * RANGE]; };       // of the groups' ranges, and of the next ones
// By 128 threads, a barrier for all of the CTA in it: the ranges of `block`, the columns of `part` of `parts`.
template <typename T, int BYTES, int RANGE>
__device__ __forceinline__ void sum_ranges(Sorted<RANGE>& sorted, int tid, int block, int part, int parts, const T* __restrict__ dy, const EoScratch& S, int n, int V, int pieces,
                                           int tpr, int range, int d, float scale, T* __restrict__ dtable) {
  using R = typename Raw<T, BYTES>::type;
  using P = Piece<T, BYTES>;
  auto& ids = sorted.ids;
  auto& toks = sorted.toks;
  R* out = reinterpret_cast<R*>(dtable);
  const int groups = 128 / tpr, group = tid / tpr, lane = tid % tpr;
  const long long r0 = (long long)block * groups;
  for (int i = tid; i < groups * (2 * range + 2); i += 128) {
    const int g = i / (2 * range + 2), e = i % (2 * range + 2);
    const long long at = (r0 + g) * range - 1 + e;
    ids[g][e] = at >= 0 && at < n ? S.id[at] : V;                  // (V: takes no gradient)
    if (e >= 1 && e <= 2 * range) toks[g][e - 1] = at < n ? S.tok[at] : 0;
  }
  const long long r = r0 + group;
  const int before_last = r >= 1 && (r - 1) * range - 1 >= 0 && (r - 1) * range - 1 < n ? S.id[(r - 1) * range - 1] : V;
  __syncthreads();
  const int* id = ids[group] + 1;                                  // id[-1], id[range ..]: the neighbours
  const int* tok = toks[group];
  int begin = 0, end = 0;                                          // rows that are added here; those that take a gradient come first
  while (end < range && id[end] < V) end += end + ROWS_AHEAD <= range && id[end + ROWS_AHEAD - 1] < V ? ROWS_AHEAD : 1;
  if (id[-1] == id[0] && id[range] != id[0] && before_last != id[0])        // the range before finishes what it began
    while (begin < end && id[begin] == id[-1]) ++begin;
  const int last = id[range - 1];
  if (last < V && last == id[range] && !(id[0] == last && id[-1] == last)) {      // begins here and goes on:
    if (id[2 * range] != last) {                                   // to be finished here,
      while (id[end] == last) ++end;
    } else if (lane == 0 && part == 0) {                           // or over a whole range and further, to be joined
      S.joins[atomicAdd(S.join_count, 1)] = make_int2((int)r, last);
    }
  }
  const R* g = reinterpret_cast<const R*>(dy);
  for (int c = part * tpr + lane; c < pieces; c += parts * tpr) {
    P acc;
    bool fresh = true, first = begin == 0;
    for (int i0 = begin; i0 < end; i0 += ROWS_AHEAD) {
      R raw[ROWS_AHEAD];
#pragma unroll
      for (int u = 0; u < ROWS_AHEAD; ++u)
        if (i0 + u < end) raw[u] = g[(long long)tok[i0 + u] * pieces + c];
#pragma unroll
      for (int u = 0; u < ROWS_AHEAD; ++u) {
        const int i = i0 + u;
        if (i >= end) break;
        const P x = unpack<T, BYTES>(raw[u]);
#pragma unroll
        for (int w = 0; w < P::N; ++w) acc.v[w] = fresh ? x.v[w] : acc.v[w] + x.v[w];
        fresh = id[i + 1] != id[i];
        if (!fresh && i + 1 < end) continue;
        const bool before = first && id[-1] == id[i];
        if (before || !fresh) {
          float* p = S.part + ((size_t)r * 2 + !before) * d + c * P::N;
#pragma unroll
          for (int w = 0; w < P::N; ++w) p[w] = acc.v[w];
        } else {
          out[(long long)id[i] * pieces + c] = pack<T, BYTES>(acc, scale);
        }
        first = false;
      }
    }
  }
}

template <typename T, int BYTES>
__global__ void __launch_bounds__(128)
embedding_sum_kernel(const T* __restrict__ dy, EoScratch S, int n, int V, int pieces, int tpr, int range, int d, float scale, T* __restrict__ dtable, int range_ctas) {
  rte::after_previous_grid();
  using R = typename Raw<T, BYTES>::type;
  __shared__ Sorted<MAX_RANGE> sorted;
  if ((int)blockIdx.x >= range_ctas) {
    R* out = reinterpret_cast<R*>(dtable);
    const int tid = threadIdx.x, groups = 128 / tpr, group = tid / tpr, lane = tid % tpr;
    int* named = sorted.ids[0];                                    // (MAX_RANGE of them)
    const long long v0 = (long long)ZERO_ROWS * (blockIdx.x - range_ctas);
    if (tid < ZERO_ROWS) {
      const int v = (int)min(v0 + tid, (long long)V), at = below(S.id, n, v);
      named[tid] = at < n && S.id[at] == v;
    }
    __syncthreads();
    for (int r = group; r < ZERO_ROWS && v0 + r < V; r += groups)
      if (!named[r])
        for (int c = blockIdx.y * tpr + lane; c < pieces; c += gridDim.y * tpr) out[(v0 + r) * pieces + c] = R{};
    return;
  }
  sum_ranges<T, BYTES, MAX_RANGE>(sorted, threadIdx.x, blockIdx.x, blockIdx.y, gridDim.y, dy, S, n, V, pieces, tpr, range, d, scale, dtable);
}

// What several ranges have of an id, added in their order: eight warps each take a run of neighbouring ranges, then the warps' sums.
constexpr int JOIN_WARPS = 8, JOIN_COLUMNS = 128;
using JoinSums = float[JOIN_WARPS][JOIN_COLUMNS];
// (CTAs and parts unsigned, as a grid's are: with int the gradient of 131072 x 2048 takes 244 us for 241.)
template <typename T>
__device__ __forceinline__ void join_ranges(JoinSums& sum, unsigned cta, unsigned ctas, unsigned part, unsigned parts, const EoScratch& S, int n, int range, int d,
                                            float scale, T* __restrict__ dtable) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int joins = *S.join_count;
  for (int j = cta; j < joins; j += ctas) {
    const int2 join = S.joins[j];
    const int r = join.x, v = join.y;
    // how many ranges behind r + 1 begin with the id: leaps of 1024, 32 and one range, a lane each, asked for at once
    const auto begins = [&](long long q) { const long long at = (r + 1 + q) * (long long)range; return at < n && S.id[at] == v; };
    int m = 0;
    bool near = begins(lane + 1), mid = begins(32LL * (lane + 1)), far = begins(1024LL * (lane + 1));
    int c = __popc(__ballot_sync(0xffffffffu, far));
    while (c == 32) {
      m += 32 * 1024;
      c = __popc(__ballot_sync(0xffffffffu, begins(m + 1024LL * (lane + 1))));
    }
    m += c * 1024;
    if (m > 0) mid = begins(m + 32LL * (lane + 1));
    c = __popc(__ballot_sync(0xffffffffu, mid));                   // (fewer than 32: range m + 1024 does not)
    m += c * 32;
    if (m > 0) near = begins(m + lane + 1);
    m += __popc(__ballot_sync(0xffffffffu, near)) + 1;             // r + 1 .. r + m
    const int first = int((long long)m * warp / JOIN_WARPS), last = int((long long)m * (warp + 1) / JOIN_WARPS);
    for (int c0 = part * JOIN_COLUMNS; c0 < d; c0 += parts * JOIN_COLUMNS) {
      const bool mine = tid < JOIN_COLUMNS && c0 + tid < d;
      const float begun = mine ? S.part[((size_t)r * 2 + 1) * d + c0 + tid] : 0.f;
      float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int q = first; q < last; ++q)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (c0 + lane + 32 * u < d) a[u] += S.part[(size_t)(r + 1 + q) * 2 * d + c0 + lane + 32 * u];
#pragma unroll
      for (int u = 0; u < 4; ++u) sum[warp][lane + 32 * u] = a[u];
      __syncthreads();
      if (mine) {
        float s = begun;
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; ++w) s += sum[w][tid];
        dtable[(long long)v * d + c0 + tid] = (T)(s * scale);
      }
      __syncthreads();
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(32 * JOIN_WARPS)
embedding_join_kernel(EoScratch S, int n, int range, int d, float scale, T* __restrict__ dtable) {
  rte::after_previous_grid();
  __shared__ JoinSums sum;
  join_ranges<T>(sum, blockIdx.x, gridDim.x, blockIdx.y, gridDim.y, S, n, range, d, scale, dtable);
}

// ---------------------------------------------------------------- few tokens: one launch
// The same three steps by one cluster, a barrier between them, with the same bits; the other clusters write the zeros, of rows that no token
// names.  Three launches were half of the host's time that such a gradient took beside the autograd engine's own.
constexpr int FEW = ONE_CTAS * SORT_THREADS, FEW_RANGE = 8, FEW_ROWS = 4096;
// The first row from r on whose bit is set, `rows` if none is; every warp for itself.
__device__ __forceinline__ int next_named(const uint32_t* named, int r, int rows) {
  const int lane = threadIdx.x & 31;
  for (int w0 = r / 32; w0 * 32 < rows; w0 += 32) {
    const int w = w0 + lane;
    uint32_t bits = w * 32 < rows ? named[w] : 0;
    if (w == r / 32) bits &= 0xffffffffu << (r % 32);
    const uint32_t some = __ballot_sync(0xffffffffu, bits);
    if (some == 0) continue;
    const int first = __ffs(some) - 1;
    return (w0 + first) * 32 + __ffs(__shfl_sync(0xffffffffu, bits, first)) - 1;
  }
  return rows;
}
// Zeros in a CTA's share of the rows, run by run between those that a token names.
__device__ __forceinline__ void zero_unnamed(const int64_t* __restrict__ ids, int n, int V, long long padding, char* table, long long row_bytes, int cta, int ctas) {
  __shared__ uint32_t named[FEW_ROWS / 32];
  const int tid = threadIdx.x;
  const long long each = ((long long)V + ctas - 1) / ctas, last = min((cta + 1) * each, (long long)V);
  for (long long v0 = cta * each; v0 < last; v0 += FEW_ROWS) {
    const int rows = (int)min(last - v0, (long long)FEW_ROWS);
    for (int i = tid; i < FEW_ROWS / 32; i += SORT_THREADS) named[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += SORT_THREADS) {
      const long long v = ids[i];
      if (v >= v0 && v < v0 + rows && v != padding) atomicOr(&named[(v - v0) / 32], 1u << ((v - v0) % 32));
    }
    __syncthreads();
    for (int r = 0; r < rows;) {
      const int to = next_named(named, r, rows);
      if (to > r) fill({table + (v0 + r) * row_bytes, (to - r) * row_bytes}, 0, 1);
      r = to + 1;
    }
    __syncthreads();
  }
}
template <typename T, int BYTES>
__global__ void __cluster_dims__(ONE_CTAS, 1, 1) __launch_bounds__(SORT_THREADS)
embedding_few_kernel(const int64_t* __restrict__ ids, int n, int V, long long padding, EoScratch S, int passes, int bits, const T* __restrict__ dy, int pieces, int tpr, int d,
                     float scale, T* __restrict__ dtable, int* status) {
  rte::after_previous_grid();
  const int tid = threadIdx.x;
  if (blockIdx.x >= ONE_CTAS) return zero_unnamed(ids, n, V, padding, reinterpret_cast<char*>(dtable), (long long)d * sizeof(T), blockIdx.x - ONE_CTAS, gridDim.x - ONE_CTAS);
  sort_one<1>(ids, n, V, padding, S, passes, bits, status);
  __shared__ Sorted<FEW_RANGE> sorted[2];                          // (each half of the CTA adds for itself)
  const int half = tid / 128, rank = blockIdx.x, ranges = (n + FEW_RANGE - 1) / FEW_RANGE, groups = 128 / tpr;
  const int parts = (pieces + tpr - 1) / tpr, units = (ranges + groups - 1) / groups * parts;
  for (int u = 2 * rank; u < units; u += 2 * ONE_CTAS) {
    __syncthreads();
    sum_ranges<T, BYTES, FEW_RANGE>(sorted[half], tid % 128, (u + half) / parts, (u + half) % parts, parts, dy, S, n, V, pieces, tpr, FEW_RANGE, d, scale, dtable);
  }
  if (ranges <= 2) return;
  static_assert(SORT_THREADS == 32 * JOIN_WARPS, "the join takes all threads");
  cg::this_cluster().sync();
  __shared__ JoinSums sum;
  join_ranges<T>(sum, rank, ONE_CTAS, 0, 1, S, n, FEW_RANGE, d, scale, dtable);
}

// ---------------------------------------------------------------- launches
bool type_ok(int type) { return type == RTE_TYPE_BF16 || type == RTE_TYPE_F16 || type == RTE_TYPE_F32; }
// the widest pieces that every row of the two tensors starts on
int piece_bytes(const void* a, const void* b, long long row_bytes) {
  const uintptr_t all = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | (uintptr_t)row_bytes;
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

// (in 64 bits: d is at most 2^30, a row's bytes are not; the kernels' columns, a grid's width beyond the last, stay within an int)
template <typename T, int BYTES> int pieces_of(int d) { return int((long long)d * (int)sizeof(T) / BYTES); }

template <typename T, int BYTES>
void launch_fwd(const int64_t* ids, long long n, const void* table, int V, int d, float scale, void* out, int* status, cudaStream_t st) {
  const int pieces = pieces_of<T, BYTES>(d), tpr = threads_per_row(pieces);
  const long long ctas = rte::ceil_div64(n, (long long)(128 / tpr) * TOKENS_AHEAD);
  const int columns = (int)min((long long)rte::ceil_div(pieces, tpr), rte::ceil_div64(148 * 8, ctas));      // few tokens: a CTA per 128 pieces
  rte::launch(embedding_fwd_kernel<T, BYTES>, dim3((unsigned)min(ctas, 148LL * 64), columns), 128, 0, st, ids, n, static_cast<const T*>(table), V, pieces, tpr, scale,
              static_cast<T*>(out), status);
}
template <typename T, int BYTES>
void launch_sum(const void* dy, const EoScratch& s, int n, int V, int d, float scale, void* dtable, bool filled, cudaStream_t st) {
  const int pieces = pieces_of<T, BYTES>(d), tpr = max(threads_per_row(pieces), MIN_TPR), range = range_of(n), ranges = rte::ceil_div(n, range);
  const int range_ctas = rte::ceil_div(ranges, 128 / tpr);
  const dim3 grid(range_ctas + (filled ? 0 : rte::ceil_div(V, ZERO_ROWS)), (unsigned)min(rte::ceil_div(pieces, tpr), 64));
  rte::launch(embedding_sum_kernel<T, BYTES>, grid, 128, 0, st, static_cast<const T*>(dy), s, n, V, pieces, tpr, range, d, scale, static_cast<T*>(dtable), range_ctas);
  if (ranges > 2) {                                                // (an id that is joined fills a range between two others)
    const int tiles = min(rte::ceil_div(d, JOIN_COLUMNS), 64);
    rte::launch(embedding_join_kernel<T>, dim3(min(ranges - 2, rte::ceil_div(148 * 8, tiles)), tiles), 32 * JOIN_WARPS, 0, st, s, n, range, d, scale, static_cast<T*>(dtable));
  }
}

constexpr int FILL_CTAS = 16 * 148;

// Whether one cluster adds the rows too: up to FEW tokens whose sums are little more than one round of the cluster's (FEW_UNITS runs of 128 threads), and no more
// table rows than come to 64 a CTA of zeros (named rows end its runs).  The host's time of a gradient's launches 8.5 us -> 3.4; us on the device,
// three launches | one: 24 x 1518 fp16 of 1206 10.1 | 10.2, 181 x 160 fp32 of 41627 11.8 | 9.8, 128 x 1024 bf16 of 32768 15.5 | 14.0, 16 x 1024 of 32768 13.6 |
// 13.9, 2048 x 8 of 131072 16.6 | 18.0; beyond the rule 500 x 1024 of 32768 17.1 | 23.7, 2048 x 8 of 10^6 18 | 50.
constexpr int FEW_UNITS = 24;
template <typename T, int BYTES>
bool launch_few(const int64_t* ids, int n, const void* dy, const EoScratch& s, int V, int d, float scale, long long padding, void* dtable, int* status, cudaStream_t st) {
  if (n > FEW || V > 64 * FILL_CTAS) return false;
  static_assert(FEW < 8192, "ranges of FEW_RANGE rows");
  const int pieces = pieces_of<T, BYTES>(d), tpr = max(threads_per_row(pieces), MIN_TPR), range_ctas = rte::ceil_div(rte::ceil_div(n, FEW_RANGE), 128 / tpr);
  if ((long long)range_ctas * rte::ceil_div(pieces, tpr) > FEW_UNITS) return false;
  const Digits dg = digits_of(V, ONE_BITS);
  // a CTA of zeros per 32 KB or 64 rows
  const long long zeros = max((long long)V * d * (int)sizeof(T) / 32768, (long long)V / 64);
  const int fills = (int)min((zeros / ONE_CTAS + 1) * ONE_CTAS, (long long)FILL_CTAS);
  rte::launch(embedding_few_kernel<T, BYTES>, ONE_CTAS + fills, SORT_THREADS, 0, st, ids, n, V, padding, s, dg.passes, dg.bits, static_cast<const T*>(dy), pieces, tpr, d, scale,
              static_cast<T*>(dtable), status);
  return true;
}

// id and tok sorted; `table` (NULL: not) filled with zeros on the way, by FILL_CTAS CTAs in each launch (33333 x 770 fp32 of 50257, the whole
// gradient, 1 | 2 | 7 | 16 of them per SM: 91 | 78 | 72 | 70 us), a pass's share twice that of the count, which is done sooner.
void launch_sort(const int64_t* ids, int n, int V, long long padding, const EoScratch& s, char* table, long long table_bytes, int* status, cudaStream_t st) {
  const bool one = n <= SORT_ONE;
  const Digits dg = digits_of(V, one ? ONE_BITS : SORT_BITS);
  const int fills = table ? FILL_CTAS : 0, shares = one ? 1 : 1 + 2 * dg.passes;
  const long long share = table ? rte::ceil_div64(rte::ceil_div64(table_bytes, shares), 256) * 256 : 0;
  auto slice = [&](int from, int to) { const long long at = min(from * share, table_bytes); return Fill{table + at, min(to * share, table_bytes) - at}; };
  if (one) {
    rte::launch(embedding_sort_kernel, ONE_CTAS + fills, SORT_THREADS, 0, st, ids, n, V, padding, s, dg.passes, dg.bits, slice(0, 1), status);
    return;
  }
  const int span = sort_span(n), ctas = rte::ceil_div(n, span);
  rte::launch(embedding_count_kernel, ctas + fills, SORT_THREADS, 0, st, ids, n, V, padding, s, dg.passes, dg.bits, span, ctas, slice(0, 1), status);
  const int *id = nullptr, *tok = nullptr;
  for (int p = 0; p < dg.passes; ++p) {
    const bool to_first = (dg.passes - 1 - p) % 2 == 0;
    int *id_out = to_first ? s.id : s.id2, *tok_out = to_first ? s.tok : s.tok2;
    const auto place = sort_each(n) == 4 ? embedding_place_kernel<4> : embedding_place_kernel<8>;
    rte::launch(place, ctas + fills, SORT_THREADS, 0, st, ids, id, tok, id_out, tok_out, s.hist, n, V, padding, p, dg.passes, dg.bits, span, ctas,
                slice(1 + 2 * p, 3 + 2 * p));
    id = id_out;
    tok = tok_out;
  }
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
  RTE_CHECK_ARG(ids && table && out && type_ok(type) && n > 0 && V > 0 && d > 0 && d <= RTE_EMBEDDING_MAX_COLUMNS);
  const int bytes = piece_bytes(table, out, (long long)d * (type == RTE_TYPE_F32 ? 4 : 2));
  if (type == RTE_TYPE_F32 && bytes < 4) return RTE_ERR_ALIGNMENT;
#define CALL(T, B) launch_fwd<T, B>(ids, n, table, V, d, scale, out, status, ST(stream))
  BY_PIECE(type, bytes, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}

extern "C" int64_t rte_embedding_bwd_scratch(int64_t n, int32_t d) {
  if (n <= 0 || d <= 0 || n > RTE_EMBEDDING_MAX_TOKENS || d > RTE_EMBEDDING_MAX_COLUMNS) return 0;
  return (int64_t)eo_layout(nullptr, n, d, nullptr);
}

extern "C" int rte_embedding_bwd(const int64_t* ids, int64_t n, const void* dy, int32_t type, int32_t V, int32_t d, float scale, int64_t padding_idx, void* dtable,
                                 void* scratch, int64_t scratch_bytes, int32_t* status, rte_stream_t stream) {
  RTE_CHECK_ARG(ids && dy && dtable && scratch && type_ok(type) && n > 0 && n <= RTE_EMBEDDING_MAX_TOKENS && V > 0 && V < 0x7fffffff && d > 0 &&
                d <= RTE_EMBEDDING_MAX_COLUMNS);
  if (scratch_bytes < rte_embedding_bwd_scratch(n, d)) return RTE_ERR_SCRATCH_CAPACITY;
  if (reinterpret_cast<uintptr_t>(scratch) & 15) return RTE_ERR_ALIGNMENT;
  const int bytes = piece_bytes(dy, dtable, (long long)d * (type == RTE_TYPE_F32 ? 4 : 2));
  if (type == RTE_TYPE_F32 && bytes < 4) return RTE_ERR_ALIGNMENT;
  EoScratch s;
  eo_layout(static_cast<char*>(scratch), n, d, &s);
  // Rows that no token names: with no more tokens than rows the whole table is filled beside the sort, and the named rows are written again; else
  // they are looked for beside the sums (us, filled ahead | looked for: 33333 x 770 fp32 of 50257 69 | 89, 60000 x 2048 bf16 of 131072 188 | 186, 131072 x
  // 2048 of 131072 241 | 244).
  const bool fill_ahead = n <= V;
  bool few = false;
#define CALL(T, B) few = launch_few<T, B>(ids, (int)n, dy, s, V, d, scale, padding_idx, dtable, status, ST(stream))
  BY_PIECE(type, bytes, CALL);
#undef CALL
  if (few) {
    RTE_LAUNCH_CHECK();
    return RTE_OK;
  }
  launch_sort(ids, (int)n, V, padding_idx, s, fill_ahead ? static_cast<char*>(dtable) : nullptr, (long long)V * d * (type == RTE_TYPE_F32 ? 4 : 2), status, ST(stream));
#define CALL(T, B) launch_sum<T, B>(dy, s, (int)n, V, d, scale, dtable, fill_ahead, ST(stream))
  BY_PIECE(type, bytes, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}
