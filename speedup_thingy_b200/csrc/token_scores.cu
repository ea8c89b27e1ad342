// Scores of tokens under a row of logits, and their gradients (operator table: k_token_logprobs, k_distill_topk).
//
// With m = max_j x_j, c = 1 / temperature, s = sum_j exp((x_j - m) c):
//   log p_j = (x_j - m) c - ln s,   H = ln s - (1 / s) sum_j exp((x_j - m) c) (x_j - m) c      (two sums of terms of one sign)
//   d log p_i / d x_j = c (1[i = j] - p_j),   d H / d x_j = -c p_j (log p_j + H)
// Distillation from a teacher of whom a list of tokens is known, q_i on the listed ids and r on all others together:
//   L = T^2 [ sum_i q_i (ln q_i - log p_i) + r (ln r - ln P) ],  P = sum of p over the others,  M = sum q + r
//   d L / d x_j = T (M p_j - q_j) on the list, T p_j (M - r / P) elsewhere
//
// Logits of the type's lowest value are ordinary numbers; -inf has probability zero and adds nothing to H.  A row of nothing but -inf
// has no distribution: log probabilities -inf, H = 0, no gradient.  NaN or +inf make a row's results NaN.
//
// Forward walks a row once, 16 bytes at a time, with a running maximum per thread; the threads' (and, where rows are few, a
// cluster's) sums meet at the end, and with them the lists of the largest logits that were noted on the way.  Backward is a pass over
// the row from its kept maximum and sum.  Both are bound by HBM as far as they are simple: gradients of 8192 x 32768 bf16 171 us
// = 6290 GB/s, sums and entropy alone 91 us = 5900 GB/s (8.8 K instructions a row at 67 % of the issue slots are close behind; the
// special-function unit could do no more than 1.37 times HBM's rate of bf16 logits).  Lists and the rest of a distillation are bound by their
// instructions: 64 alternatives make it 157 us, a list of 64 left out of the sum 123.

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "rte_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int TS_MAX_LIST = RTE_TOKEN_LIST_MAX;
// Forward's CTAs on an SM: 24 to 40 warps are in flight, a thread has 80, 48 or 64 registers.  (With 48, lists spill up to 260 bytes; ten CTAs | eight with 64
// registers, us, 32 alternatives of 2048 bf16 columns: 256 rows 6.6 | 6.2, 1000 10.8 | 8.8, 2900 19.3 | 19.9, none: 2.7 | 2.8, 4.65 | 4.25, 7.9 | 8.3.)
__host__ __device__ constexpr int min_ctas(int nt, int u) { return nt == 32 ? 24 : nt == 256 ? 4 : u == 4 ? 10 : 8; }
constexpr int TS_MAX_V = 0x7fffff00;           // (columns and what is added to them stay within an int)
constexpr float LN2 = 0.693147180559945309f;
constexpr double LOG2E = 1.44269504088896340736, LN2_D = 0.693147180559945309417;
constexpr float FAR = 0x1p27f;                 // exponents (in powers of two) beyond this are taken the careful way
constexpr float LOW = -1e30f;                  // the least logit that enters an entropy's products: far beyond FAR at any temperature
constexpr float MIN_T = 1e-6f, MAX_T = 1e6f;   // temperatures: LOW is then within fp32 after scaling
// Distillation above this temperature has its sums and its listed columns' gradients in 64 bits: the loss is T^2 times a divergence that falls
// as T^-2, so that an error of 1e-7 in a row's logarithm, fp32's, is one of T^2 1e-7 in a loss of order one.  The second pass over the row is bound
// by instructions (71 a logit, 81 % of the issue slots; the fp64 pipe 41 %): 8192 x 32768 bf16, 64 listed, us forward | backward at T = 8 and above it
// 104 | 170 and 502 | 236, with the rest 125 | 168 and 629 | 229, which is why lower temperatures, where that error is below 1e-5, go without.
constexpr float HOT_T = 8.f;

__device__ __forceinline__ float exp2_fast(float t) {            // relative error up to 2^-22.5, 0 below -126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

// Two fp32 values in one register pair, one instruction for both.
struct Two {
  unsigned long long v;
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ float lo() const { return __uint_as_float((uint32_t)v); }
  __device__ __forceinline__ float hi() const { return __uint_as_float((uint32_t)(v >> 32)); }
};
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c.v) : "l"(a.v), "l"(b.v)); return c; }
__device__ __forceinline__ Two add2(Two a, Two b) { asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v)); return a; }

__device__ __forceinline__ float max_nan(float a, float b) {     // NaN where either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---------------------------------------------------------------- 16 bytes of a row
template <typename T> struct Vec;              // N values; max: NaN where one of them is; unpack_low: at least LOW
template <> struct Vec<float> {
  static constexpr int SHIFT = 0;                       // low bits that a value's key does not use
  static constexpr int N = 4;
  static constexpr uint32_t NONE = 0xff800000u;                  // -inf
  static __device__ __forceinline__ void unpack(const uint4& r, float (&x)[4]) {
    x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y); x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ float max(const uint4& r) {
    return max_nan(max_nan(__uint_as_float(r.x), __uint_as_float(r.y)), max_nan(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
  static __device__ __forceinline__ void unpack_low(const uint4& r, float (&x)[4]) {
    unpack(r, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = max_nan(x[i], LOW);
  }
  static __device__ __forceinline__ float to_f(float v) { return v; }
  static __device__ __forceinline__ float from_f(float v) { return v; }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int SHIFT = 16;
  static constexpr int N = 8;
  static constexpr uint32_t NONE = 0xff80ff80u;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  static __device__ __forceinline__ float max(const uint4& r) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    return make_uint4(rte::pack_bf16x2(x[0], x[1]), rte::pack_bf16x2(x[2], x[3]), rte::pack_bf16x2(x[4], x[5]), rte::pack_bf16x2(x[6], x[7]));
  }
  static __device__ __forceinline__ void unpack_low(const uint4& r, float (&x)[8]) {
    const __nv_bfloat162 low = __float2bfloat162_rn(LOW);
    uint4 q;
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<__nv_bfloat162*>(&q)[i] = __hmax2_nan(reinterpret_cast<const __nv_bfloat162*>(&r)[i], low);
    unpack(q, x);
  }
  static __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Vec<__half> {
  static constexpr int SHIFT = 13;
  static constexpr int N = 8;
  static constexpr uint32_t NONE = 0xfc00fc00u;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&x)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 f = __half22float2(h[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
  }
  static __device__ __forceinline__ float max(const uint4& r) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint4 pack(const float (&x)[8]) {
    uint4 r;
    __half2* h = reinterpret_cast<__half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    return r;
  }
  static __device__ __forceinline__ void unpack_low(const uint4& r, float (&x)[8]) {
    unpack(r, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = max_nan(x[i], LOW);
  }
  static __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
};

// A row as 16-byte pieces: piece v holds the columns [v * N - off, (v + 1) * N - off), so that all but the first and the last lie
// whole inside the row, on 16 bytes.  Columns outside the row read as -inf.
template <typename T>
struct Row {
  static constexpr int N = Vec<T>::N;
  const T* x;
  int V, off, pieces;
  __device__ __forceinline__ Row(const T* row, int V_) : x(row), V(V_), off(int(reinterpret_cast<uintptr_t>(row) & 15) / (int)sizeof(T)), pieces((V_ + off + N - 1) / N) {}
  __device__ __forceinline__ int column(int v) const { return v * N - off; }
  __device__ __forceinline__ bool whole(int v) const { const int c = column(v); return c >= 0 && c + N <= V; }
  __device__ __forceinline__ uint4 load(int v) const {
    const int c = column(v);
    if (c >= 0 && c + N <= V) return __ldg(reinterpret_cast<const uint4*>(x + c));
    uint4 r = make_uint4(Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE);
    T* t = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < N; ++i) if (c + i >= 0 && c + i < V) t[i] = x[c + i];
    return r;
  }
  __device__ __forceinline__ float at(int column) const { return Vec<T>::to_f(x[column]); }
};

// ---------------------------------------------------------------- sums of exponentials
// Exponents are kept in powers of two relative to R = top * c, top the largest logit, c = log2(e) / T: t = x c - R in one fused step,
// whose rounded R shifts every t of a row alike, by up to half a step of R, and is taken out again at the end.  Below |R| = FAR that is 4 at
// most; from 2^31 on it could be 128, where 2^t is infinite or 0.  So a row whose R is beyond FAR is summed again with t = (x - top) c, and
// a tile whose largest logit lies below -2 FAR is left out (`masked`): with ordinary logits in the row it counts nothing (FAR
// powers of two less), without any the row is summed again, and no running R that anything was summed with is lower.  Logits below LOW count
// as LOW where t is multiplied (t is then finite, so that t 2^t is 0 as 2^t is); a row of nothing but -inf has the sum 0.
struct Sums { float top, R, s, e; };           // largest logit, reference, sum of 2^t, sum of t 2^t
__device__ __forceinline__ float reference(float top, float c) { return fmaxf(top, LOW) * c; }
__device__ __forceinline__ bool far(float top, float c) { return !(fabsf(top * c) < FAR); }
__device__ __forceinline__ bool masked(float top, float c) { return top * c <= -2.f * FAR; }
__device__ __forceinline__ Sums no_sums(float c) { return {-INFINITY, LOW * c, 0.f, 0.f}; }
__device__ __forceinline__ void move_to(Sums& a, float R) {      // the same sums relative to R >= a.R
  const float d = a.R - R, f = exp2_fast(d);
  a.e = f * (a.e + d * a.s);
  a.s *= f;
  a.R = R;
}
__device__ __forceinline__ float weighted(float t) { return fmaxf(t, -1e4f); }       // (t 2^t is 0 where t = -inf)

template <int NT>
__device__ __forceinline__ Sums block_sums(Sums a, float c, Sums* red) {  // red: NT / 32 of them in shared memory; every thread gets the result
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (q == 1) {
      if (NT == 32) break;
      __syncthreads();
      if (lane == 0) red[warp] = a;
      __syncthreads();
      a = lane < NT / 32 ? red[lane] : no_sums(c);
    }
    move_to(a, rte::warp_max(a.R));
    a.top = rte::warp_max(a.top);
    a.s = rte::warp_sum(a.s);
    a.e = rte::warp_sum(a.e);
  }
  return a;
}
__device__ __forceinline__ bool careful(const Sums& a, float c) { return a.top != -INFINITY && far(a.top, c); }

// The exponent of a logit relative to the row's largest, as forward formed it; p = 2^(t - l2) with l2 as forward kept it.
struct Near {
  float c, R;
  __device__ __forceinline__ Near(float top, float c_) : c(c_), R(reference(top, c_)) {}
  __device__ __forceinline__ float operator()(float x) const { return fmaf(x, c, -R); }
};
struct Far {
  float top, c;
  __device__ __forceinline__ Far(float top_, float c_) : top(top_), c(c_) {}
  __device__ __forceinline__ float operator()(float x) const { return (x - top) * c; }
};

// ---------------------------------------------------------------- the largest logits of a row
// Order of the alternatives: value, NaN above all, then the lower column.  Larger keys come first.
__device__ __forceinline__ uint32_t value_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);                            // (-0 = 0)
  return v != v ? 0xfffffffeu : (b & 0x80000000u ? ~b : b | 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(float v, int column) { return (unsigned long long)value_key(v) << 32 | (uint32_t)~column; }
__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t u = uint32_t(key >> 32);
  return u == 0xfffffffeu ? __uint_as_float(0x7fffffffu) : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// The k largest logits lie in the k pieces (16 bytes of the row) whose own largest logits come first, equal ones by the lower piece: every
// other piece holds only what k logits come before.  So the search goes over pieces, an eighth or a quarter of the columns: those that
// reach a bound are noted, the bound is the k-th of what has been seen (the first one the k-th of the threads' largest, so that a
// few more than k pieces of a tile pass), and only in the end the columns of the last k pieces, and a few more, are ordered.
__host__ __device__ constexpr int slack_of(int k) { return (k < 64 ? k : 64) + 32 + (k < 64 ? 0 : k & 1); }       // (k + slack is even)
struct TopK {                                            // in shared memory, sized by k: `shared_bytes`
  struct Head { unsigned long long bound; int count, keep, from, pad[3]; };
  Head& h;
  unsigned long long *kept, *piece;                      // [k + slack], [cap]: value | ~piece; from piece + k + slack on, in the end: value | ~column
  uint32_t* top;                                         // [threads]
  int k, cap;
  // a round's pieces behind twice what is kept; behind the pieces kept all their columns, which is also what 8 slices keep
  static __host__ __device__ int most(int k) { return k + slack_of(k); }
  static __host__ __device__ int cap_of(int k, int round) { return max(round + 2 * most(k), 9 * most(k)); }
  static size_t shared_bytes(int k, int nt, int round) { return sizeof(Head) + 8 * ((size_t)most(k) + cap_of(k, round)) + 4 * ((size_t)nt + round); }
  float* tops;                                           // [round]: the largest of every piece of a round, each its thread's own
  __device__ __forceinline__ TopK(unsigned char* at, int k_, int nt, int round)
      : h(*reinterpret_cast<Head*>(at)), kept(reinterpret_cast<unsigned long long*>(at + sizeof(Head))), piece(kept + most(k_)),
        top(reinterpret_cast<uint32_t*>(piece + cap_of(k_, round))), k(k_), cap(cap_of(k_, round)), tops(reinterpret_cast<float*>(top + nt)) {}
  __device__ __forceinline__ unsigned long long* column_list() const { return piece + most(k); }
};
// Tiles whose pieces' maxima are kept before they are looked through: 512, 1024 and 2048 pieces.
__host__ __device__ constexpr int round_tiles(int nt, int u) { return nt == 32 ? 4 : nt == 128 && u == 4 ? 2 : 1; }

template <int NT> __device__ __forceinline__ void sync() { if (NT == 32) __syncwarp(); else __syncthreads(); }
template <int NT> __device__ __forceinline__ int sync_or(int v) { return NT == 32 ? __any_sync(0xffffffffu, v) : __syncthreads_or(v); }

// Room in a list for the n keys that each lane brings: where this lane's begin, and the count behind the warp's (0: it brings
// none).  One atomic per warp: 32 lanes on one counter would take their turns.
__device__ __forceinline__ int2 reserve(int* count, int n) {
  const int lane = threadIdx.x & 31;
  if (!__any_sync(0xffffffffu, n)) return make_int2(0, 0);
  int upto = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += v; }
  int at = 0;
  if (lane == 31) at = atomicAdd(count, upto);
  at = __shfl_sync(0xffffffffu, at, 31);
  return make_int2(at + upto - n, at + __shfl_sync(0xffffffffu, upto, 31));
}
__device__ __forceinline__ void append(unsigned long long* to, int* count, bool mine, unsigned long long key) {
  const uint32_t who = __ballot_sync(0xffffffffu, mine);
  if (who == 0) return;
  int at = 0;
  if ((threadIdx.x & 31) == 0) at = atomicAdd(count, __popc(who));
  at = __shfl_sync(0xffffffffu, at, 0);
  if (mine) to[at + __popc(who & ((1u << (threadIdx.x & 31)) - 1))] = key;
}

// The largest bound that at least k (at most k + slack, unless equal keys forbid) of n keys reach; one warp.  Its lanes hold HELD keys each
// (0: none, below every bound), more are read from keys[i * STEP], i from 32 * HELD on.  SHIFT: the low bits of a key that say
// nothing (a 16-bit logit's are all 0 or all 1), not searched.
template <int SHIFT, int STEP, int HELD>
__device__ __forceinline__ uint32_t search_bound(const uint32_t (&held)[HELD], const uint32_t* keys, int n, int k, int slack, int* reach) {
  const int lane = threadIdx.x & 31;
  uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll
  for (int u = 0; u < HELD; ++u) {
    lo = min(lo, held[u] - 1);                           // (the predecessor of 0 is above all)
    hi = max(hi, held[u]);
  }
  for (int i = lane + 32 * HELD; i < n; i += 32) { lo = min(lo, keys[i * STEP] - 1); hi = max(hi, keys[i * STEP]); }
  lo = (__reduce_min_sync(0xffffffffu, lo) + 1) >> SHIFT;
  hi = (__reduce_max_sync(0xffffffffu, hi) >> SHIFT) + 1;            // (no key is ~0)
  int at_lo = n;
  for (int probe = 0; hi - lo > 1 && at_lo > k + slack; ++probe) {
    uint32_t mid = lo + (hi - lo) / 2;
    if (probe < 6) {                                     // halfway between the values first: logits lie about a mean, their keys about zero
      const uint32_t half = value_key(0.5f * key_value((unsigned long long)lo << (32 + SHIFT)) + 0.5f * key_value((unsigned long long)(hi - 1) << (32 + SHIFT))) >> SHIFT;
      if (half > lo && half < hi) mid = half;
    }
    const uint32_t bound = mid << SHIFT;
    int c = 0;
#pragma unroll
    for (int u = 0; u < HELD; ++u) c += held[u] >= bound;
    for (int i = lane + 32 * HELD; i < n; i += 32) c += keys[i * STEP] >= bound;
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= k) { lo = mid; at_lo = c; } else hi = mid;
  }
  *reach = at_lo;
  return lo << SHIFT;
}
template <int SHIFT, int STEP, int HELD>
__device__ __forceinline__ uint32_t warp_bound(const uint32_t* keys, int n, int k, int slack, int* reach) {
  uint32_t held[HELD];
#pragma unroll
  for (int u = 0; u < HELD; ++u) {
    const int i = (threadIdx.x & 31) + 32 * u;
    held[u] = i < n ? keys[i * STEP] : 0;
  }
  return search_bound<SHIFT, STEP, HELD>(held, keys, n, k, slack, reach);
}

// A bound that at least k and at most k + slack of n distinct keys reach, n > k + slack; one warp.
template <int SHIFT>
__device__ __noinline__ unsigned long long warp_bound64(const unsigned long long* keys, int n, int k, int slack) {
  const int lane = threadIdx.x & 31;
  int reach;
  const uint32_t* values = reinterpret_cast<const uint32_t*>(keys) + 1;
  const uint32_t value = n <= 128 ? warp_bound<SHIFT, 2, 4>(values, n, k, slack, &reach)
                                  : n <= 256 ? warp_bound<SHIFT, 2, 8>(values, n, k, slack, &reach) : warp_bound<SHIFT, 2, 16>(values, n, k, slack, &reach);
  if (reach <= k + slack) return (unsigned long long)value << 32;
  int above = 0;                                         // many equal values at the end: the lowest of their columns
  uint32_t same = 0;                                     // (their key, with the bits that were not searched)
  for (int i = lane; i < n; i += 32)
    if (uint32_t(keys[i] >> 32) >> SHIFT == value >> SHIFT) same = uint32_t(keys[i] >> 32);
  same = __reduce_max_sync(0xffffffffu, same);
  for (int i = lane; i < n; i += 32) above += uint32_t(keys[i] >> 32) > same;
  const int want = k - __reduce_add_sync(0xffffffffu, above);
  unsigned long long lo = 0, hi = 1ull << 32;
  int at_lo = reach - (k - want);
  while (hi - lo > 1 && at_lo > want + slack) {
    const unsigned long long mid = lo + (hi - lo) / 2;
    int c = 0;
    for (int i = lane; i < n; i += 32) c += uint32_t(keys[i] >> 32) == same && uint32_t(keys[i]) >= mid;
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= want) { lo = mid; at_lo = c; } else hi = mid;
  }
  return (unsigned long long)same << 32 | lo;
}

// kept = those of n > k + slack keys that reach a bound which k to k + slack of them reach; keep: how many.  Everyone is past writing them.
template <int NT, int SHIFT>
__device__ __forceinline__ void thin(TopK& S, const unsigned long long* keys, int n, int slack) {
  if (threadIdx.x < 32) {
    const unsigned long long b = warp_bound64<SHIFT>(keys, n, S.k, slack);
    if (threadIdx.x == 0) { S.h.bound = b > S.h.bound ? b : S.h.bound; S.h.keep = 0; }
  }
  sync<NT>();
  const unsigned long long b = S.h.bound;
  for (int i = threadIdx.x; (i & ~31) < n; i += NT) {
    const unsigned long long key = i < n ? keys[i] : 0;
    append(S.kept, &S.h.keep, i < n && key >= b, key);
  }
  sync<NT>();
}

// Looks through a round: notes those of this thread's pieces (tops[j * NT + tid]: the largest of piece first + j * NT, below `end`) that
// reach the bound.  all: the largest of them.  Leaves room for another round where one follows.
template <int NT, int COUNT, int SHIFT>
__device__ __forceinline__ void note(TopK& S, float all, int first, int end, bool start) {
  constexpr int round = NT * COUNT;
  const int tid = threadIdx.x;
  const int have = first < end ? min((end - first + NT - 1) / NT, COUNT) : 0;
  if (start) {
    uint32_t b = 0;
    int reach;
    if (NT == 32) {                                      // a warp knows all of its pieces
      const int n = min(end - (first - tid), round);
      uint32_t key[COUNT];
#pragma unroll
      for (int j = 0; j < COUNT; ++j) key[j] = j < have ? value_key(S.tops[j * NT + tid]) : 0;
      if (n > S.k) b = search_bound<SHIFT, 1, COUNT>(key, nullptr, n, S.k, S.k / 8, &reach);
      if (tid == 0) { S.h.count = 0; S.h.bound = (unsigned long long)b << 32; }
    } else {
      const int n = min(end - (first - tid), NT);        // threads with a piece
      S.top[tid] = value_key(all);
      if (tid == 0) S.h.count = 0;
      __syncthreads();
      if (tid < 32) {
        if (n > S.k) b = warp_bound<SHIFT, 1, NT / 32>(S.top, n, S.k, S.k / 8, &reach);
        if (tid == 0) S.h.bound = (unsigned long long)b << 32;
      }
    }
    sync<NT>();
  }
  const unsigned long long bound = S.h.bound;
  const float least = key_value(bound);                  // (NaN: no bound, or NaN is)
  uint32_t mine = 0;
#pragma unroll
  for (int j = 0; j < COUNT; ++j)
    if (!(S.tops[j * NT + tid] < least)) mine |= 1u << j;
  mine &= (1u << have) - 1;
  int2 at = reserve(&S.h.count, __popc(mine));
  const bool full = at.y > S.cap - round;
  while (mine) {
    const int j = __ffs(mine) - 1;
    mine &= mine - 1;
    S.piece[at.x++] = order_key(S.tops[j * NT + tid], first + j * NT);
  }
  if (first - tid + round >= end || !sync_or<NT>(full)) return;      // (the count itself may grow while others still look)
  const int n = S.h.count;
  thin<NT, SHIFT>(S, S.piece, n, slack_of(S.k));
  const int keep = S.h.keep;
  for (int i = tid; i < keep; i += NT) S.piece[i] = S.kept[i];
  if (tid == 0) S.h.count = keep;
  sync<NT>();
}
// The keys at `from` (0: kept, 1: column_list), if they are many thinned out into `kept`.
template <int NT, int SHIFT>
__device__ __forceinline__ void shorten(TopK& S) {
  sync<NT>();
  const int n = S.h.count;
  if (n > TopK::most(S.k)) {                             // (what is left is ordered by counting, n^2 comparisons)
    thin<NT, SHIFT>(S, S.column_list(), n, S.k / 8 + 8);
    if (threadIdx.x == 0) S.h.from = 0;
  } else if (threadIdx.x == 0) {
    S.h.keep = n;
    S.h.from = 1;
  }
  sync<NT>();
}
// In the end: `keep` columns at `from` among which the row's (the slice's) k largest logits are, no more than k + slack.
template <typename T, int NT>
__device__ __forceinline__ void columns(TopK& S, const Row<T>& row) {
  constexpr int N = Vec<T>::N;
  sync<NT>();
  int n = S.h.count;
  const unsigned long long* from = S.piece;
  if (n > TopK::most(S.k)) {
    thin<NT, Vec<T>::SHIFT>(S, S.piece, n, slack_of(S.k));
    n = S.h.keep;
    from = S.kept;
  }
  const unsigned long long bound = S.h.bound & 0xffffffff00000000ull;     // (of k pieces' largest: k columns reach its value)
  sync<NT>();
  if (threadIdx.x == 0) { S.h.count = 0; S.h.bound = bound; }
  sync<NT>();
  const float least = key_value(bound);
  for (int i0 = threadIdx.x; (i0 & ~31) < n; i0 += 2 * NT) {                     // two pieces a thread, both requested at once
    uint4 raw[2];
    int c[2];
    uint32_t mine[2] = {0, 0};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (i0 + u * NT >= n) continue;
      const int v = (int)~(uint32_t)from[i0 + u * NT];
      raw[u] = row.load(v);
      c[u] = row.column(v);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (i0 + u * NT >= n) continue;
      float x[N];
      Vec<T>::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < N; ++j) if (!(x[j] < least)) mine[u] |= 1u << j;
      if (c[u] < 0 || c[u] + N > row.V)
        for (int j = 0; j < N; ++j) if (c[u] + j < 0 || c[u] + j >= row.V) mine[u] &= ~(1u << j);
    }
    int2 at = reserve(&S.h.count, __popc(mine[0]) + __popc(mine[1]));
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (mine[u] == 0) continue;
      float x[N];
      Vec<T>::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (mine[u] >> j & 1) S.column_list()[at.x++] = order_key(x[j], c[u] + j);
    }
  }
  shorten<NT, Vec<T>::SHIFT>(S);
}

// ---------------------------------------------------------------- one pass over a row's pieces [begin, end)
// OUTSIDE: the columns of `id` (-1: none) are left out; `bits`: a bit per column of MAP_TILES tiles, in shared memory.
constexpr int MAP_TILES = 8;
template <typename T, int NT, int U, bool ENTROPY, bool TOP, bool OUTSIDE>
__device__ __forceinline__ Sums stream(const Row<T>& row, int begin, int end, float c, TopK* top_k, const int* id, int ids, uint32_t* bits) {
  constexpr int N = Vec<T>::N, TILE = NT * U;
  const int tid = threadIdx.x;
  Sums a = no_sums(c);
  constexpr int ROUND = round_tiles(NT, U);
  int in_round = 0;
  float round_top = 0.f;
  for (int tile = begin; tile < end; tile += TILE) {
    const int first = tile + tid;
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      raw[u] = first + u * NT < end ? row.load(first + u * NT) : make_uint4(Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE);
    if (OUTSIDE) {
      const int in_map = (tile - begin) % (TILE * MAP_TILES);
      if (in_map == 0) {
        sync<NT>();
        for (int i = tid; i < TILE * MAP_TILES * N / 32; i += NT) bits[i] = 0;
        sync<NT>();
        for (int i = tid; i < ids; i += NT) {
          const int at = id[i] + row.off - tile * N;
          if (id[i] >= 0 && at >= 0 && at < TILE * MAP_TILES * N) atomicOr(&bits[at >> 5], 1u << (at & 31));
        }
        sync<NT>();
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = (in_map + u * NT + tid) * N;
        const uint32_t listed = bits[at / 32] >> (at % 32) & ((1u << N) - 1);
        if (listed) {
          uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const uint32_t mask = N == 4 ? 0xffffffffu : i % 2 ? 0xffff0000u : 0x0000ffffu;
            if (listed >> i & 1) w[i * 4 / N] = (w[i * 4 / N] & ~mask) | (Vec<T>::NONE & mask);
          }
          raw[u] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    float top[U], all = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) { top[u] = Vec<T>::max(raw[u]); all = max_nan(all, top[u]); }
    if (all > a.top) a.top = all;
    if (!masked(all, c)) {                                       // (NaN is not)
      const float R = fmaxf(a.R, reference(a.top, c));
      if (R > a.R) move_to(a, R);
      const Two cc(c, c), negR(-a.R, -a.R);
      Two s(0.f, 0.f), e(0.f, 0.f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[N];
        if (ENTROPY) Vec<T>::unpack_low(raw[u], x);
        else Vec<T>::unpack(raw[u], x);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
          const Two t = fma2(Two(x[i], x[i + 1]), cc, negR), p(exp2_fast(t.lo()), exp2_fast(t.hi()));
          s = add2(s, p);
          if (ENTROPY) e = fma2(p, t, e);
        }
      }
      a.s += s.lo() + s.hi();
      if (ENTROPY) a.e += e.lo() + e.hi();
    }
    if (TOP) {
#pragma unroll
      for (int u = 0; u < U; ++u) top_k->tops[(in_round * U + u) * NT + tid] = top[u];
      round_top = in_round == 0 ? all : max_nan(round_top, all);
      if (++in_round == ROUND || tile + TILE >= end) {
        const int before = (in_round - 1) * TILE;
        note<NT, U * ROUND, Vec<T>::SHIFT>(*top_k, round_top, first - before, end, tile - before == begin);
        in_round = 0;
      }
    }
  }
  return a;
}

// The sums of a row whose reference is out of range (`careful`): relative to its largest logit, which is not -inf.
template <typename T, int NT, bool OUTSIDE>
__device__ __noinline__ Sums sums_far(const Row<T> row, int begin, int end, float top, float c, const int* id, int ids, Sums* red) {
  float s = 0.f, e = 0.f;
  for (int j = max(row.column(begin), 0) + (int)threadIdx.x; j < min(row.column(end), row.V); j += NT) {
    bool out = false;
    if (OUTSIDE) for (int i = 0; i < ids; ++i) out |= id[i] == j;
    if (out) continue;
    const float t = (row.at(j) - top) * c, p = exp2_fast(t);
    s += p;
    e = fmaf(p, weighted(t), e);
  }
  Sums a = {top, 0.f, s, e};
  a = block_sums<NT>(a, c, red);
  return a;
}

__device__ __forceinline__ double warp_sum_double(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The sum of exp((x - top) / T) over a row's pieces [begin, end) in 64 bits, top not -inf; OUTSIDE and `bits` as in `stream`.
template <typename T, int NT, int U, bool OUTSIDE>
__device__ __noinline__ double sum_hot(const Row<T> row, int begin, int end, float top, double inv_t, const int* id, int ids, uint32_t* bits, double* red) {
  constexpr int N = Vec<T>::N, SPAN = NT * U * MAP_TILES;
  const int tid = threadIdx.x;
  double s = 0;
  for (int at = begin; at < end; at += SPAN) {
    if (OUTSIDE) {
      sync<NT>();
      for (int i = tid; i < SPAN * N / 32; i += NT) bits[i] = 0;
      sync<NT>();
      for (int i = tid; i < ids; i += NT) {
        const int bit = id[i] + row.off - at * N;
        if (id[i] >= 0 && bit >= 0 && bit < SPAN * N) atomicOr(&bits[bit >> 5], 1u << (bit & 31));
      }
      sync<NT>();
    }
    for (int v = at + tid; v < min(at + SPAN, end); v += NT) {
      const int bit = (v - at) * N;
      const uint32_t listed = OUTSIDE ? bits[bit / 32] >> (bit % 32) : 0;
      float x[N];
      Vec<T>::unpack(row.load(v), x);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (!(listed >> i & 1)) s += exp(((double)x[i] - top) * inv_t);
    }
  }
  s = warp_sum_double(s);
  if (NT == 32) return s;
  __syncthreads();
  if (tid % 32 == 0) red[tid / 32] = s;
  __syncthreads();
  return warp_sum_double(tid % 32 < NT / 32 ? red[tid % 32] : 0.);
}

// ---------------------------------------------------------------- forward
// A cluster of C CTAs per row, each with a slice of its pieces; rank 0 joins what they found.  us (k = 0 | listed): 8192 x 32768 bf16
// 91 | 157 (64), 8192 x 2048 11.0 | 31 (32), 61 x 131072 fp32 12 | 19 (8), 1 x 50257 bf16 4.1 | 9.0 (20), 1531 x 50257 31.
template <typename T, int NT, int U, bool TOP>
__global__ void __launch_bounds__(NT, min_ctas(NT, U))
token_logprobs_kernel(const T* __restrict__ logits, long long ld, const int64_t* __restrict__ tokens, long long ignore, float c, float inv_t, int k, float* __restrict__ logprob,
                      float* __restrict__ entropy, float* __restrict__ top_lp, int64_t* __restrict__ top_ids, float2* __restrict__ stats, int V, int C, int* status) {
  rte::after_previous_grid();
  extern __shared__ __align__(16) unsigned char dyn[];
  TopK top(dyn, k, NT, NT * U * round_tiles(NT, U));                                     // (there is none without TOP)
  __shared__ Sums red[NT / 32];
  __shared__ Sums mine;
  const long long row_at = blockIdx.x / C;
  const int rank = blockIdx.x % C, tid = threadIdx.x;
  const long long tok = tokens[row_at];
  if (tok < 0 || tok >= V || tok == ignore) {
    if (rank == 0) {
      if (tok != ignore && status && tid == 0) atomicExch(status, RTE_DEV_INDEX_OUT_OF_RANGE);
      if (tid == 0) {
        logprob[row_at] = 0.f;
        entropy[row_at] = 0.f;
        if (stats) stats[row_at] = make_float2(0.f, -INFINITY);
      }
      for (int i = tid; i < k; i += NT) { top_lp[row_at * k + i] = 0.f; top_ids[row_at * k + i] = -1; }
    }
    return;
  }
  const Row<T> row(logits + row_at * ld, V);
  float target = 0.f;
  if (rank == 0 && tid == 0) target = row.at((int)tok);
  const int per = (row.pieces + C - 1) / C, begin = min(rank * per, row.pieces), end = min(begin + per, row.pieces);
  Sums a = stream<T, NT, U, true, TOP, false>(row, begin, end, c, &top, nullptr, 0, nullptr);
  a = block_sums<NT>(a, c, red);
  if (TOP) {
    if (begin < end) columns<T, NT>(top, row);
    else if (tid == 0) { top.h.keep = 0; top.h.from = 0; top.h.bound = 0; }
  }
  if (C > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) mine = a;
    cluster.sync();
    a = no_sums(c);
    for (int r = 0; r < C; ++r) {
      Sums b = *cluster.map_shared_rank(&mine, r);
      const float R = fmaxf(a.R, b.R);
      move_to(a, R);
      move_to(b, R);
      a.top = fmaxf(a.top, b.top);
      a.s += b.s;
      a.e += b.e;
    }
    if (careful(a, c)) {                                            // (all CTAs of the cluster see the same sums)
      const Sums b = sums_far<T, NT, false>(row, begin, end, a.top, c, nullptr, 0, red);
      cluster.sync();
      if (tid == 0) mine = b;
      cluster.sync();
      a = b;
      a.s = a.e = 0.f;
      for (int r = 0; r < C; ++r) { const Sums* o = cluster.map_shared_rank(&mine, r); a.s += o->s; a.e += o->e; }
    }
    if (TOP && rank == 0) {                                      // the others' lists behind this CTA's
      int n = top.h.keep;
      if (!top.h.from) for (int i = tid; i < n; i += NT) top.column_list()[i] = top.kept[i];
      for (int r = 1; r < C; ++r) {
        const TopK::Head* h = cluster.map_shared_rank(&top.h, r);
        const unsigned long long* list = cluster.map_shared_rank(h->from ? top.column_list() : top.kept, r);
        const int m = h->keep;
        for (int i = tid; i < m; i += NT) top.column_list()[n + i] = list[i];
        n += m;
      }
      cluster.sync();                                            // (the others leave)
      if (tid == 0) top.h.count = n;
      shorten<NT, Vec<T>::SHIFT>(top);
    } else {
      cluster.sync();
    }
    if (rank != 0) return;
  } else if (careful(a, c)) {
    a = sums_far<T, NT, false>(row, begin, end, a.top, c, nullptr, 0, red);
  }
  const bool none = a.s == 0.f;                                  // nothing but -inf
  const int n = TOP ? top.h.keep : 0;
  const unsigned long long* list = TOP && top.h.from ? top.column_list() : top.kept;
  if (tid >= max(n, 1)) return;
  // ln of the sum relative to the largest logit: without the rounding of R
  float ln_s = logf(a.s) - LN2 * (far(a.top, c) ? 0.f : fmaf(a.top, c, -a.R));
  if (ln_s < 0.f) ln_s = 0.f;                                    // (the largest logit alone makes it 0; no log probability above 0)
  const auto log_p = [&](float x) { return none ? -INFINITY : (x - a.top) * inv_t - ln_s; };
  if (tid == 0) {
    logprob[row_at] = log_p(target);
    // H = ln s - sum t 2^t / s, relative to the same R
    const float H = LN2 * (log2f(a.s) - a.e / a.s);
    entropy[row_at] = none || H < 0.f ? 0.f : H;
    if (stats) stats[row_at] = make_float2(a.top, none ? -INFINITY : log2f(a.s));
  }
  for (int i = tid; i < n; i += NT) {                            // the list's order: how many keys come before
    const unsigned long long key = list[i];
    int before = 0;                                              // (a bitonic network of one warp instead: 183 us for 159, 35 for 31)
#pragma unroll 4
    for (int j = 0; j + 1 < n; j += 2) {                         // (the lists start on 16 bytes)
      const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(list + j);
      before += two.x > key;
      before += two.y > key;
    }
    if (n & 1) before += list[n - 1] > key;
    if (before >= k) continue;
    top_ids[row_at * k + before] = (int)~(uint32_t)key;
    top_lp[row_at * k + before] = log_p(key_value(key));
  }
}

// As above; the teacher's list and the student's logits on it are requested ahead of the row.  us: 8192 x 32768 bf16, 64 and the rest 123 (4360
// GB/s; the listed columns' bits are a quarter of its instructions), 1999 x 50257 fp16, 50, renormalised, 30 % of the rows empty 34, 256 x 2048 fp32 5.1.
// stats of a row, eight floats: for the columns outside the list (all, without TAIL) their largest logit, log2 of their sum and what
// their share of it is multiplied by; M (0: no gradient); the list's max, ln of its sum; the row's largest logit, log2 of its sum.  HOT: of
// the last four ln of the row's sum over M in 64 bits (two of them), the row's largest logit, whether the list stays as it is (TAIL).
template <typename T, int NT, int U, bool TAIL, bool HOT>
__global__ void __launch_bounds__(NT, HOT ? min_ctas(NT, U) / 2 : min_ctas(NT, U))
distill_topk_kernel(const T* __restrict__ logits, long long ld, const float* __restrict__ teacher, const int64_t* __restrict__ ids, int k, float c, double temp,
                    float* __restrict__ loss, float4* __restrict__ stats, int V, int C, int* status) {
  rte::after_previous_grid();
  __shared__ __align__(16) int id[TS_MAX_LIST];
  __shared__ float listed[TS_MAX_LIST];                          // the student's logits on the list
  __shared__ uint32_t bits[TAIL ? NT * U * MAP_TILES * Vec<T>::N / 32 : 1];
  __shared__ Sums red[NT / 32];
  __shared__ Sums mine;
  __shared__ double red_hot[HOT ? NT / 32 : 1], mine_hot;
  const long long row_at = blockIdx.x / C;
  const int rank = blockIdx.x % C, tid = threadIdx.x;
  const float* t = teacher + row_at * k;
  const Row<T> row(logits + row_at * ld, V);
  bool any = false;
  float tmax = -INFINITY;                                        // the list's largest
  for (int i = tid; i < k; i += NT) {
    const long long v = ids[row_at * k + i];
    if (v >= V && status) atomicExch(status, RTE_DEV_INDEX_OUT_OF_RANGE);
    id[i] = v < 0 || v >= V ? -1 : (int)v;
    if (id[i] < 0) continue;
    any |= TAIL || t[i] != -INFINITY;
    listed[i] = row.at(id[i]);
  }
  any = __syncthreads_or(any);
  if (!any) {                                                    // (the same in all CTAs of the cluster)
    if (rank == 0 && tid == 0) {
      loss[row_at] = 0.f;
      if (stats) stats[row_at * 2] = stats[row_at * 2 + 1] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  const int per = (row.pieces + C - 1) / C, begin = min(rank * per, row.pieces), end = min(begin + per, row.pieces);
  Sums a = stream<T, NT, U, false, false, TAIL>(row, begin, end, c, nullptr, id, k, bits);
  a = block_sums<NT>(a, c, red);
  const double inv_t = 1. / temp;
  double hot = 0;                                                // HOT: the sum relative to a.top
  if (C > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) mine = a;
    cluster.sync();
    a = no_sums(c);
    for (int r = 0; r < C; ++r) {
      Sums b = *cluster.map_shared_rank(&mine, r);
      const float R = fmaxf(a.R, b.R);
      move_to(a, R);
      move_to(b, R);
      a.top = fmaxf(a.top, b.top);
      a.s += b.s;
    }
    if (HOT) {
      if (a.top != -INFINITY) hot = sum_hot<T, NT, U, TAIL>(row, begin, end, a.top, inv_t, id, k, bits, red_hot);
      if (tid == 0) mine_hot = hot;
      cluster.sync();
      hot = 0;
      for (int r = 0; r < C; ++r) hot += *cluster.map_shared_rank(&mine_hot, r);
    } else if (careful(a, c)) {
      const Sums b = sums_far<T, NT, TAIL>(row, begin, end, a.top, c, id, k, red);
      cluster.sync();
      if (tid == 0) mine = b;
      cluster.sync();
      a = b;
      a.s = 0.f;
      for (int r = 0; r < C; ++r) a.s += cluster.map_shared_rank(&mine, r)->s;
    }
    cluster.sync();                                              // (the others leave)
    if (rank != 0) return;
  } else if (HOT) {
    if (a.top != -INFINITY) hot = sum_hot<T, NT, U, TAIL>(row, begin, end, a.top, inv_t, id, k, bits, red_hot);
  } else if (careful(a, c)) {
    a = sums_far<T, NT, TAIL>(row, begin, end, a.top, c, id, k, red);
  }
  // The rest is one warp's (with all of them at it 13.4 K instructions a row of 32768 with a list of 64, now 12.2 K), and in 64 bits: a few
  // values per row, whose small differences are the loss.
  if (tid >= 32) return;
  float top = a.top;                                             // the row's largest logit
  const bool others = HOT ? hot != 0 : a.s != 0.f;
  const double shift = far(a.top, c) ? 0. : (double)a.top * c - reference(a.top, c);      // log2 of what a.s is too large by
  double s = HOT ? hot : a.s * exp2(-shift), ln_factor = 0;      // the row's sum relative to `top`; ln of what a.s is relative to less than it
  if (TAIL) {
    float m = a.top;
    for (int i = tid; i < k; i += 32) if (id[i] >= 0) m = fmaxf(m, listed[i]);
    top = rte::warp_max(m);
    double l = 0;
    if (top != -INFINITY)
      for (int i = tid; i < k; i += 32) {
        bool again = id[i] < 0;                                  // a token that an earlier slot names too counts once
        for (int j = 0; j < i; j += 4) {
          const int4 v = *reinterpret_cast<const int4*>(id + j);
          again |= v.x == id[i] || (j + 1 < i && v.y == id[i]) || (j + 2 < i && v.z == id[i]) || (j + 3 < i && v.w == id[i]);
        }
        const double d = (listed[i] - (double)top) * inv_t;
        if (!again) l += HOT ? exp(d) : expf((float)d);
      }
    l = warp_sum_double(l);
    ln_factor = others ? ((double)a.top - top) * inv_t : 0.;
    s = l + s * exp(ln_factor);
  }
  const double ln_s = log(s);
  const bool none = top == -INFINITY && s == 0;                  // nothing but -inf
  double t_shift = 0;
  if (!TAIL) {
    float m = -INFINITY;
    for (int i = tid; i < k; i += 32) if (id[i] >= 0) m = fmaxf(m, t[i]);
    tmax = rte::warp_max(m);
    double l = 0;
    for (int i = tid; i < k; i += 32) if (id[i] >= 0) l += exp((double)t[i] - tmax);
    t_shift = log(warp_sum_double(l));
  }
  double M = 0, L = 0;
  for (int i = tid; i < k; i += 32) {
    if (id[i] < 0) continue;
    const double lq = TAIL ? (double)t[i] : (double)t[i] - tmax - t_shift, q = exp(lq);
    M += q;
    if (q != 0) L += q * (lq - (none ? -INFINITY : (listed[i] - (double)top) * inv_t - ln_s));
  }
  M = warp_sum_double(M);
  L = warp_sum_double(L);
  if (tid != 0) return;
  double P = 1;                                                  // the others' probability
  if (TAIL) {
    const double r = (HOT ? hot > 0 : a.s > 0.f) ? fmax(0., 1 - M) : 0., ln_out = ln_factor + (HOT ? log(hot) : log((double)a.s) - shift * LN2_D) - ln_s;
    P = exp(ln_out);
    if (r > 0) L += r * (log(r) - ln_out);
    M += r;
    P = M * P - r;                                               // (what the others' gradient is in proportion to)
  }
  loss[row_at] = float(L * temp * temp);
  if (!stats) return;
  // 2^-l2 of a sum relative to the rounded reference that backward forms again: the others' among themselves, and the row's
  stats[row_at * 2] = make_float4(others ? a.top : 0.f, others ? HOT ? float(log2(hot) + shift) : log2f(a.s) : 0.f, !others ? 0.f : TAIL ? (float)P : (float)M,
                                  none ? 0.f : (float)M);
  if (HOT) {
    const double A = ln_s - log(M);
    stats[row_at * 2 + 1] = make_float4(__int_as_float(__double2hiint(A)), __int_as_float(__double2loint(A)), top, TAIL ? 1.f : 0.f);
    return;
  }
  const double l2 = ln_s * LOG2E + (far(top, c) ? 0. : (double)top * c - reference(top, c));
  stats[row_at * 2 + 1] = make_float4(TAIL ? 0.f : tmax, (float)t_shift, top, (float)l2);
}

// ---------------------------------------------------------------- backward
// A CTA per NT * U pieces of a row: what all columns get first, from the row's saved maximum and sum; then its first warp writes the
// listed columns again.  32 registers, so that an SM holds 2048 threads: with 48, scores 181 us and distillation 208 instead of 171 and 168 (8192 x
// 32768 bf16, 6290 and 6400 GB/s); 1531 x 50257, whose rows start anywhere, 48 us = 6360 GB/s.
template <typename T, int NT, int U>
struct Slice {
  Row<T> row;
  T* dx;
  bool even;                                                     // logits and gradient lie alike on 16 bytes
  int first;                                                     // piece
  __device__ __forceinline__ Slice(const T* x, T* dx_, int V, int part)
      : row(x, V), dx(dx_), even(((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx_)) & 15) == 0), first(part * NT * U + threadIdx.x) {}
  __device__ __forceinline__ bool holds(long long column, int part) const {
    const long long v = (column + row.off) / Vec<T>::N - (long long)part * NT * U;
    return column >= 0 && column < row.V && v >= 0 && v < NT * U;
  }
  __device__ __forceinline__ void store(int v, const float (&y)[Vec<T>::N]) const {
    const int c = row.column(v);
    if (even && row.whole(v)) { *reinterpret_cast<uint4*>(dx + c) = Vec<T>::pack(y); return; }
#pragma unroll
    for (int i = 0; i < Vec<T>::N; ++i) if (c + i >= 0 && c + i < row.V) dx[c + i] = Vec<T>::from_f(y[i]);
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) if (first + u * NT < row.pieces) raw[u] = row.load(first + u * NT);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (first + u * NT >= row.pieces) break;
      float x[Vec<T>::N];
      Vec<T>::unpack(raw[u], x);
#pragma unroll
      for (int i = 0; i < Vec<T>::N; ++i) x[i] = f(x[i]);
      store(first + u * NT, x);
    }
  }
  __device__ __forceinline__ void zero() const {
    const float y[Vec<T>::N] = {};
    for (int u = 0; u < U; ++u) if (first + u * NT < row.pieces) store(first + u * NT, y);
  }
};

template <typename T, int NT, int U>
__global__ void __launch_bounds__(NT, NT == 32 ? 24 : 2048 / NT)
token_logprobs_bwd_kernel(const T* __restrict__ logits, long long ld, const int64_t* __restrict__ tokens, float c, float inv_t, int k, const int64_t* __restrict__ top_ids,
                          const float2* __restrict__ stats, const float* __restrict__ entropy, const float* __restrict__ g_lp, const float* __restrict__ g_h,
                          const float* __restrict__ g_top, T* __restrict__ dlogits, int V, int parts) {
  rte::after_previous_grid();
  const long long row_at = blockIdx.x / parts, tok = tokens[row_at];
  const int part = blockIdx.x % parts, tid = threadIdx.x;
  const float2 st = stats[row_at];
  const Slice<T, NT, U> slice(logits + row_at * ld, dlogits + row_at * V, V, part);
  if (tok < 0 || tok >= V || st.y == -INFINITY) return slice.zero();          // (an ignored row's sum was kept as 0 too)
  const float g = g_lp ? g_lp[row_at] : 0.f, gh = g_h ? g_h[row_at] : 0.f;
  float all = 0.f;
  for (int i = tid & 31; g_top && i < k; i += 32) all += g_top[row_at * k + i];        // (every warp for itself)
  all = g + rte::warp_sum(all);
  // dx = -p (all + gh (ln p + H)) / T
  const float a = -(all + gh * entropy[row_at]) * inv_t, b = -gh * LN2 * inv_t;
  const auto write = [&](auto exponent) {
    const auto base = [&](float x) {
      const float l = exponent(x) - st.y;
      return exp2_fast(l) * fmaf(b, weighted(l), a);
    };
    slice.each(base);
    sync<NT>();
    if (tid >= 32) return;
    bool target_done = !g_lp || !slice.holds(tok, part);
    for (int i = tid; g_top && i - tid < k; i += 32) {
      const long long j = i < k ? top_ids[row_at * k + i] : -1;
      const bool target = j == tok, mine = slice.holds(j, part);
      if (mine) dlogits[row_at * V + j] = Vec<T>::from_f(base(slice.row.at((int)j)) + (g_top[row_at * k + i] + (target ? g : 0.f)) * inv_t);
      target_done |= __any_sync(0xffffffffu, target && mine);
    }
    if (!target_done && tid == 0) dlogits[row_at * V + tok] = Vec<T>::from_f(base(slice.row.at((int)tok)) + g * inv_t);
  };
  if (far(st.x, c)) write(Far(st.x, c));
  else write(Near(st.x, c));
}

template <typename T, int NT, int U, bool HOT>
__global__ void __launch_bounds__(NT, HOT ? 1024 / NT < 16 ? 1024 / NT : 16 : NT == 32 ? 24 : 2048 / NT)
distill_topk_bwd_kernel(const T* __restrict__ logits, long long ld, const float* __restrict__ teacher, const int64_t* __restrict__ ids, int k, float c, float temp,
                        const float4* __restrict__ stats, const float* __restrict__ dloss, T* __restrict__ dlogits, int V, int parts) {
  rte::after_previous_grid();
  constexpr int MAP = NT * U * Vec<T>::N / 32;
  __shared__ int id[TS_MAX_LIST];
  __shared__ std::conditional_t<HOT, double, float> q[TS_MAX_LIST];
  __shared__ uint32_t map[MAP];                                  // a bit per column of the slice
  const long long row_at = blockIdx.x / parts;
  const int part = blockIdx.x % parts, tid = threadIdx.x;
  const float4 st = stats[row_at * 2];
  const Slice<T, NT, U> slice(logits + row_at * ld, dlogits + row_at * V, V, part);
  if (st.w == 0.f) return slice.zero();
  const float scale = dloss[row_at] * temp;
  {
    const float outside = scale * st.z;
    if (far(st.x, c)) { const Far t(st.x, c); slice.each([&](float x) { return exp2_fast(t(x) - st.y) * outside; }); }
    else { const Near t(st.x, c); slice.each([&](float x) { return exp2_fast(t(x) - st.y) * outside; }); }
  }
  sync<NT>();
  if (tid >= 32) return;
  const float4 list = stats[row_at * 2 + 1];
  const float inside = scale * st.w;
  const bool is_far = far(list.z, c);
  const Far from(list.z, c);
  const Near near(list.z, c);
  double A = 0, L = 0;                                           // HOT: M p = exp((x - top) / T - A), q = exp(t - L)
  if (HOT) {
    A = __hiloint2double(__float_as_int(list.x), __float_as_int(list.y));
    if (list.w == 0.f) {                                         // the renormalised list's logarithm, as forward formed it
      float m = -INFINITY;
      for (int i = tid; i < k; i += 32) { const long long j = ids[row_at * k + i]; if (j >= 0 && j < V) m = fmaxf(m, teacher[row_at * k + i]); }
      m = rte::warp_max(m);
      double l = 0;
      for (int i = tid; i < k; i += 32) { const long long j = ids[row_at * k + i]; if (j >= 0 && j < V) l += exp((double)teacher[row_at * k + i] - m); }
      L = m + log(warp_sum_double(l));
    }
  }
  for (int i = tid; i < MAP; i += 32) map[i] = 0;
  __syncwarp();
  int n = 0;                                                     // the slots that name a column of this slice, in their order
  bool twice = false;
  for (int i = tid; i - tid < k; i += 32) {
    const long long j = i < k ? ids[row_at * k + i] : -1;
    const bool mine = slice.holds(j, part);
    const uint32_t who = __ballot_sync(0xffffffffu, mine);
    if (mine) {
      const int at = n + __popc(who & ((1u << tid) - 1));
      id[at] = (int)j;
      if (HOT) q[at] = exp(teacher[row_at * k + i] - L);
      else q[at] = expf(teacher[row_at * k + i] - list.x - list.y);
      const int bit = (int)j + slice.row.off - part * NT * U * Vec<T>::N;
      twice |= atomicOr(&map[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1;
    }
    n += __popc(who);
  }
  twice = __any_sync(0xffffffffu, twice);
  for (int i = tid; i < n; i += 32) {
    bool again = false;                                          // a token named by several slots: the first of them writes
    auto sum = q[i];
    if (twice) {
      sum = 0;
      for (int j = 0; j < n; ++j)
        if (id[j] == id[i]) { again |= j < i; sum += q[j]; }
    }
    if (again) continue;
    const float x = slice.row.at(id[i]);
    if (HOT) dlogits[row_at * V + id[i]] = Vec<T>::from_f(float(scale * (exp(((double)x - list.z) / temp - A) - sum)));
    else dlogits[row_at * V + id[i]] = Vec<T>::from_f(exp2_fast((is_far ? from(x) : near(x)) - list.w) * inside - scale * sum);
  }
}

// ---------------------------------------------------------------- launches
template <typename K, typename... A>
void launch_cluster(K kernel, long long ctas, int nt, size_t smem, int C, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(nt);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = C > 1 ? 2 : 1;
  (void)cudaLaunchKernelEx(&cfg, kernel, args...);               // (an error stays pending for RTE_LAUNCH_CHECK)
}

// CTAs per row: as many (up to 8) as come to ten on an SM, with a tile of pieces each; to four where their lists have to be joined too, two if the rows
// are not that long.  us, 1 | 2 | 4 | 8 per row: 300 x 50257 bf16 13.1 | 12.4 | 10.3 | 15.6, 700 x 50257 21 | 15.6 | 18.8 | 30; with lists 61 x 131072 fp32
// 42 | 29 | 20 | 19, 150 x 32768 bf16 11.2 | 13.7, 1000 x 32768 31 | 38 | 55 | 103.
int cluster_of(long long rows, int pieces, int tile, bool lists) {
  int C = 1;
  while (C < 8 && rows * C * 2 <= (!lists ? 10 : pieces > 8 * tile ? 4 : 2) * 148 && pieces > C * tile) C *= 2;
  return C;
}
// The most pieces a row of V columns has: one more where rows do not all start on 16 bytes.
int pieces_of(const void* x, int type, long long ld, int V) {
  const int size = type == RTE_TYPE_F32 ? 4 : 2, n = 16 / size;
  const bool even = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld * size % 16 == 0;
  return int(((long long)V + (even ? n - 1 : 2 * n - 2)) / n);
}

// A row of at most one tile of 32 or 128 threads is one CTA of them; longer ones are walked by 256.
// Forward, who walks a row.  Many short rows: a warp each (us, 8192 x 2048 bf16, warp | 128 threads: 10.7 | 18.5, with 32 alternatives 31 | 49;
// 16384 x 5000 41 | 57, with 32 93 | 117; 16384 x 9001 with 50 168 | 187; 16384 x 16000 108 | 98, with 50 222 | 186; 256 x 2048 3.4 | 2.7, with 32 8.3 | 6.5).  Many long ones: 128 threads (8192 x 32768 bf16, warp | 128 | 256 | 512: 119 | 97 | 105 | 151), eight loads each for
// scores, four for distillation, which has more to keep (2000 x 131072 with 64 alternatives, 4 | 8: 133 | 118; 8192 x 32768 distilled 127 | 134).
// Few long ones, where latency counts: 256 threads, eight loads each (1 x 50257 with 20 alternatives, 128 x 4 | 256 x 4 | 256 x 8: 12.8 | 10.7 | 9.2).
constexpr int MANY_SHORT = 20 * 148, MANY_LONG = 2 * 148;
#define FORWARD(T, rows, pieces, LOADS, CALL) \
  do { \
    if (pieces <= 128 || (pieces <= 1280 && rows >= MANY_SHORT)) CALL(T, 32, 4); \
    else if (pieces <= 512) CALL(T, 128, 4); \
    else if (rows >= MANY_LONG) CALL(T, 128, LOADS); \
    else CALL(T, 256, 8); \
  } while (0)
// Backward: CTAs of a warp for rows that it covers, of 128 threads for others, all 2048 of an SM (8192 x 32768 bf16, 128 | 256 threads:
// 163 | 174; 8192 x 2048, warp | 128: 17.9 | 13.7).
#define BACKWARD(T, rows, pieces, LOADS, CALL) \
  do { \
    if (pieces <= 128) CALL(T, 32, 4); \
    else CALL(T, 128, 4); \
  } while (0)
#define BY_TYPE(type, WHICH, rows, pieces, LOADS, CALL) \
  do { \
    if (type == RTE_TYPE_BF16) WHICH(__nv_bfloat16, rows, pieces, LOADS, CALL); \
    else if (type == RTE_TYPE_F16) WHICH(__half, rows, pieces, LOADS, CALL); \
    else WHICH(float, rows, pieces, LOADS, CALL); \
  } while (0)

bool temperature_ok(float t) { return t >= MIN_T && t <= MAX_T; }
bool rows_ok(const void* x, int type, int64_t ldl, int64_t rows, int64_t V) {
  return x && (type == RTE_TYPE_BF16 || type == RTE_TYPE_F16 || type == RTE_TYPE_F32) && rows > 0 && V > 0 && V <= TS_MAX_V && ldl >= 0;
}
bool on_element(const void* x, int type) { return reinterpret_cast<uintptr_t>(x) % (type == RTE_TYPE_F32 ? 4 : 2) == 0; }
float log2_scale(float temperature) { return (float)(LOG2E / temperature); }

}  // namespace

#define ST(s) static_cast<cudaStream_t>(s)

extern "C" int rte_token_logprobs_fwd(const void* logits, int32_t type, int64_t ldl, const int64_t* tokens, int64_t ignore_index, float temperature, int32_t top_k,
                                      float* logprob, float* entropy, float* top_logprobs, int64_t* top_ids, float* row_stats, int32_t rows, int32_t V, int32_t* status,
                                      rte_stream_t stream) {
  RTE_CHECK_ARG(rows_ok(logits, type, ldl, rows, V) && tokens && logprob && entropy && temperature_ok(temperature));
  RTE_CHECK_ARG(top_k >= 0 && top_k <= V && top_k <= TS_MAX_LIST && (top_k == 0 || (top_logprobs && top_ids)));
  if (!on_element(logits, type) || reinterpret_cast<uintptr_t>(row_stats) % 8) return RTE_ERR_ALIGNMENT;
  const int pieces = pieces_of(logits, type, ldl, V);
#define CALL(T, NT, U) \
  do { \
    const int C = cluster_of(rows, pieces, NT * U, top_k > 0); \
    launch_cluster(top_k > 0 ? token_logprobs_kernel<T, NT, U, true> : token_logprobs_kernel<T, NT, U, false>, (long long)rows * C, NT, \
                   top_k > 0 ? TopK::shared_bytes(top_k, NT, NT * U * round_tiles(NT, U)) : 0, C, ST(stream), static_cast<const T*>(logits), (long long)ldl, \
                   tokens, (long long)ignore_index, log2_scale(temperature), 1.f / temperature, (int)top_k, logprob, entropy, top_logprobs, \
                   top_ids, reinterpret_cast<float2*>(row_stats), (int)V, C, status); \
  } while (0)
  BY_TYPE(type, FORWARD, rows, pieces, 8, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}

extern "C" int rte_token_logprobs_bwd(const void* logits, int32_t type, int64_t ldl, const int64_t* tokens, float temperature, int32_t top_k, const int64_t* top_ids,
                                      const float* row_stats, const float* entropy, const float* g_logprob, const float* g_entropy, const float* g_top, void* dlogits,
                                      int32_t rows, int32_t V, rte_stream_t stream) {
  RTE_CHECK_ARG(rows_ok(logits, type, ldl, rows, V) && tokens && entropy && row_stats && dlogits && temperature_ok(temperature));
  RTE_CHECK_ARG(top_k >= 0 && top_k <= V && top_k <= TS_MAX_LIST && (!g_top || top_k == 0 || top_ids));
  if (!on_element(logits, type) || !on_element(dlogits, type) || reinterpret_cast<uintptr_t>(row_stats) % 8) return RTE_ERR_ALIGNMENT;
  const int pieces = pieces_of(logits, type, ldl, V);
#define CALL(T, NT, U) \
  do { \
    const int parts = rte::ceil_div(pieces, NT * U); \
    if ((long long)rows * parts > 0x7fffffff) return RTE_ERR_UNSUPPORTED; \
    rte::launch(token_logprobs_bwd_kernel<T, NT, U>, rows * parts, NT, 0, ST(stream), static_cast<const T*>(logits), ldl, tokens, log2_scale(temperature), \
                1.f / temperature, top_k, top_ids, reinterpret_cast<const float2*>(row_stats), entropy, g_logprob, g_entropy, g_top, static_cast<T*>(dlogits), V, \
                parts); \
  } while (0)
  BY_TYPE(type, BACKWARD, rows, pieces, 4, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}

extern "C" int rte_distill_topk_fwd(const void* logits, int32_t type, int64_t ldl, const float* teacher, const int64_t* ids, int32_t k, float temperature, int32_t tail,
                                    float* loss, float* row_stats, int32_t rows, int32_t V, int32_t* status, rte_stream_t stream) {
  RTE_CHECK_ARG(rows_ok(logits, type, ldl, rows, V) && teacher && ids && loss && temperature_ok(temperature));
  RTE_CHECK_ARG(k > 0 && k <= TS_MAX_LIST);
  if (!on_element(logits, type) || reinterpret_cast<uintptr_t>(row_stats) % 16) return RTE_ERR_ALIGNMENT;
  const bool hot = temperature > HOT_T;
  const int pieces = pieces_of(logits, type, ldl, V);
#define CALL(T, NT, U) \
  do { \
    const int C = cluster_of(rows, pieces, NT * U, false); \
    launch_cluster(tail ? hot ? distill_topk_kernel<T, NT, U, true, true> : distill_topk_kernel<T, NT, U, true, false> \
                        : hot ? distill_topk_kernel<T, NT, U, false, true> : distill_topk_kernel<T, NT, U, false, false>, (long long)rows * C, NT, 0, C, ST(stream), \
                   static_cast<const T*>(logits), (long long)ldl, teacher, ids, (int)k, log2_scale(temperature), (double)temperature, loss, \
                   reinterpret_cast<float4*>(row_stats), (int)V, C, status); \
  } while (0)
  BY_TYPE(type, FORWARD, rows, pieces, 4, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}

extern "C" int rte_distill_topk_bwd(const void* logits, int32_t type, int64_t ldl, const float* teacher, const int64_t* ids, int32_t k, float temperature,
                                    const float* row_stats, const float* dloss, void* dlogits, int32_t rows, int32_t V, rte_stream_t stream) {
  RTE_CHECK_ARG(rows_ok(logits, type, ldl, rows, V) && teacher && ids && row_stats && dloss && dlogits && temperature_ok(temperature));
  RTE_CHECK_ARG(k > 0 && k <= TS_MAX_LIST);
  if (!on_element(logits, type) || !on_element(dlogits, type) || reinterpret_cast<uintptr_t>(row_stats) % 16) return RTE_ERR_ALIGNMENT;
  const int pieces = pieces_of(logits, type, ldl, V);
#define CALL(T, NT, U) \
  do { \
    const int parts = rte::ceil_div(pieces, NT * U); \
    if ((long long)rows * parts > 0x7fffffff) return RTE_ERR_UNSUPPORTED; \
    rte::launch(temperature > HOT_T ? distill_topk_bwd_kernel<T, NT, U, true> : distill_topk_bwd_kernel<T, NT, U, false>, rows * parts, NT, 0, ST(stream), static_cast<const T*>(logits), ldl, teacher, ids, k, log2_scale(temperature), \
                temperature, reinterpret_cast<const float4*>(row_stats), dloss, static_cast<T*>(dlogits), V, parts); \
  } while (0)
  BY_TYPE(type, BACKWARD, rows, pieces, 4, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}
