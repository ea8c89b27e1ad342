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

#include <cuda_fp16.h>

#include "rte_common.cuh"

namespace {

constexpr int TS_THREADS = 256;
constexpr int TS_MAX_LIST = RTE_TOKEN_LIST_MAX;
constexpr float LN2 = 0.693147180559945309f, LOG2E = 1.44269504088896341f;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Order of the alternatives: value, NaN above all, then the lower column.  Larger keys come first; 0 is below and ~0 above every key.
__device__ __forceinline__ unsigned long long order_key(float v, int column) {
  const uint32_t b = __float_as_uint(v + 0.f);                            // (-0 = 0)
  const uint32_t u = v != v ? 0xfffffffeu : (b & 0x80000000u ? ~b : b | 0x80000000u);
  return (unsigned long long)u << 32 | (uint32_t)~column;
}

template <typename T>
__global__ void __launch_bounds__(TS_THREADS)
token_logprobs_kernel(const T* __restrict__ logits, long long ld, const int64_t* __restrict__ tokens, long long ignore, float inv_t, int k, float* __restrict__ logprob,
                      float* __restrict__ entropy, float* __restrict__ top_lp, int64_t* __restrict__ top_ids, float2* __restrict__ stats, int V, int* status) {
  rte::after_previous_grid();
  __shared__ float red[32];
  __shared__ unsigned long long best[32];
  const long long row = blockIdx.x, tok = tokens[row];
  const int tid = threadIdx.x;
  if (tok < 0 || tok >= V) {
    if (tok != ignore && status && tid == 0) atomicExch(status, RTE_DEV_INDEX_OUT_OF_RANGE);
    if (tid == 0) { logprob[row] = 0.f; entropy[row] = 0.f; stats[row] = make_float2(0.f, 0.f); }
    for (int i = tid; i < k; i += TS_THREADS) { top_lp[row * k + i] = 0.f; top_ids[row * k + i] = -1; }
    return;
  }
  const T* x = logits + row * ld;
  float m = -INFINITY;
  for (int j = tid; j < V; j += TS_THREADS) m = fmaxf(m, to_f(x[j]));
  m = rte::block_max(m, red);
  const float ref = m == -INFINITY ? 0.f : m;
  float s = 0.f, e1 = 0.f;
  for (int j = tid; j < V; j += TS_THREADS) {
    const float d = (to_f(x[j]) - ref) * inv_t, e = expf(d);
    s += e;
    e1 += e == 0.f ? 0.f : e * d;
  }
  s = rte::block_sum(s, red);
  e1 = rte::block_sum(e1, red);
  const float ln_s = logf(s);
  if (tid == 0) {
    logprob[row] = s == 0.f ? -INFINITY : (to_f(x[tok]) - ref) * inv_t - ln_s;
    entropy[row] = s == 0.f ? 0.f : ln_s - e1 / s;
    stats[row] = make_float2(ref, ln_s);
  }
  unsigned long long last = ~0ull;
  for (int i = 0; i < k; ++i) {
    unsigned long long mine = 0;
    for (int j = tid; j < V; j += TS_THREADS) {
      const unsigned long long key = order_key(to_f(x[j]), j);
      if (key < last && key > mine) mine = key;
    }
    for (int o = 16; o > 0; o >>= 1) { const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, o); mine = other > mine ? other : mine; }
    __syncthreads();
    if ((tid & 31) == 0) best[tid >> 5] = mine;
    __syncthreads();
    for (int w = 0; w < TS_THREADS / 32; ++w) mine = best[w] > mine ? best[w] : mine;
    last = mine;
    if (tid == 0) {
      const int j = (int)~(uint32_t)mine;
      top_ids[row * k + i] = j;
      top_lp[row * k + i] = s == 0.f ? -INFINITY : (to_f(x[j]) - ref) * inv_t - ln_s;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(TS_THREADS)
token_logprobs_bwd_kernel(const T* __restrict__ logits, long long ld, const int64_t* __restrict__ tokens, float inv_t, int k, const int64_t* __restrict__ top_ids,
                          const float2* __restrict__ stats, const float* __restrict__ entropy, const float* __restrict__ g_lp, const float* __restrict__ g_h,
                          const float* __restrict__ g_top, T* __restrict__ dlogits, int V) {
  rte::after_previous_grid();
  const long long row = blockIdx.x, tok = tokens[row];
  const float2 st = stats[row];
  T* dx = dlogits + row * V;
  const int tid = threadIdx.x;
  if (tok < 0 || tok >= V || st.y == -INFINITY) {
    for (int j = tid; j < V; j += TS_THREADS) dx[j] = from_f<T>(0.f);
    return;
  }
  const T* x = logits + row * ld;
  const float g = g_lp ? g_lp[row] : 0.f, gh = g_h ? g_h[row] : 0.f, H = entropy[row];
  float all = g;
  if (g_top) for (int i = 0; i < k; ++i) all += g_top[row * k + i];
  for (int j = tid; j < V; j += TS_THREADS) {
    const float lp = (to_f(x[j]) - st.x) * inv_t - st.y, p = expf(lp);
    float d = p == 0.f ? 0.f : -p * (all + gh * (lp + H));
    if (j == tok) d += g;
    if (g_top) for (int i = 0; i < k; ++i) if (top_ids[row * k + i] == j) d += g_top[row * k + i];
    dx[j] = from_f<T>(d * inv_t);
  }
}

// stats of a row, eight floats: max, ln s, coefficient of p outside the list, M (0: no gradient), the list's max, ln of its sum
template <typename T>
__global__ void __launch_bounds__(TS_THREADS)
distill_topk_kernel(const T* __restrict__ logits, long long ld, const float* __restrict__ teacher, const int64_t* __restrict__ ids, int k, float temp, int tail,
                    float* __restrict__ loss, float4* __restrict__ stats, int V, int* status) {
  rte::after_previous_grid();
  __shared__ float red[32];
  __shared__ int id[TS_MAX_LIST];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x;
  bool any = false;
  for (int i = tid; i < k; i += TS_THREADS) {
    const long long v = ids[row * k + i];
    if (v >= V && status) atomicExch(status, RTE_DEV_INDEX_OUT_OF_RANGE);
    id[i] = v < 0 || v >= V ? -1 : (int)v;
    any |= id[i] >= 0;
  }
  any = __syncthreads_or(any);
  double tmax = -INFINITY, tsum = 0;
  if (any && !tail) {
    any = false;
    for (int i = 0; i < k; ++i) {
      if (id[i] < 0) continue;
      tmax = fmax(tmax, (double)teacher[row * k + i]);
      any |= teacher[row * k + i] != -INFINITY;
    }
    for (int i = 0; i < k; ++i) if (id[i] >= 0) tsum += exp(teacher[row * k + i] - tmax);
  }
  if (!any) {
    if (tid == 0) { loss[row] = 0.f; stats[row * 2] = stats[row * 2 + 1] = make_float4(0.f, 0.f, 0.f, 0.f); }
    return;
  }
  const float inv_t = 1.f / temp;
  const T* x = logits + row * ld;
  float m = -INFINITY;
  for (int j = tid; j < V; j += TS_THREADS) m = fmaxf(m, to_f(x[j]));
  m = rte::block_max(m, red);
  const float ref = m == -INFINITY ? 0.f : m;
  float s = 0.f, so = 0.f;
  for (int j = tid; j < V; j += TS_THREADS) {
    bool listed = false;
    if (tail) for (int i = 0; i < k; ++i) listed |= id[i] == j;
    const float e = expf((to_f(x[j]) - ref) * inv_t);
    s += e;
    if (!listed) so += e;
  }
  s = rte::block_sum(s, red);
  so = rte::block_sum(so, red);
  if (tid == 0) {
    double M = 0, L = 0, r = 0;
    const double ln_s = log((double)s), shift = tail ? 0. : tmax + log(tsum);
    for (int i = 0; i < k; ++i) {
      if (id[i] < 0) continue;
      const double lq = teacher[row * k + i] - shift, q = exp(lq);
      M += q;
      if (q != 0) L += q * (lq - (s == 0.f ? -INFINITY : (double)((to_f(x[id[i]]) - ref) * inv_t) - ln_s));
    }
    if (tail && so > 0.f) r = fmax(0., 1 - M);
    if (r > 0) L += r * (log(r) - (log((double)so) - ln_s));
    M += r;
    loss[row] = float(L * temp * temp);
    stats[row * 2] = make_float4(ref, (float)ln_s, float(M - (r > 0 ? r * (double)s / so : 0.)), s == 0.f ? 0.f : (float)M);
    stats[row * 2 + 1] = make_float4((float)(tail ? 0. : tmax), (float)(tail ? 0. : log(tsum)), 0.f, 0.f);
  }
}

template <typename T>
__global__ void __launch_bounds__(TS_THREADS)
distill_topk_bwd_kernel(const T* __restrict__ logits, long long ld, const float* __restrict__ teacher, const int64_t* __restrict__ ids, int k, float temp,
                        const float4* __restrict__ stats, const float* __restrict__ dloss, T* __restrict__ dlogits, int V) {
  rte::after_previous_grid();
  const long long row = blockIdx.x;
  const float4 a = stats[row * 2], b = stats[row * 2 + 1];
  T* dx = dlogits + row * V;
  if (a.w == 0.f) {
    for (int j = threadIdx.x; j < V; j += TS_THREADS) dx[j] = from_f<T>(0.f);
    return;
  }
  const T* x = logits + row * ld;
  const float scale = dloss[row] * temp, inv_t = 1.f / temp;
  for (int j = threadIdx.x; j < V; j += TS_THREADS) {
    const float p = expf((to_f(x[j]) - a.x) * inv_t - a.y);
    bool listed = false;
    float q = 0.f;
    for (int i = 0; i < k; ++i)
      if (ids[row * k + i] == j) { listed = true; q += expf(teacher[row * k + i] - b.x - b.y); }
    dx[j] = from_f<T>(scale * (listed ? a.w * p - q : a.z * p));
  }
}

bool temperature_ok(float t) { return t > 0.f && t <= 1e30f && 1.f / t <= 1e30f; }
bool type_ok(int type) { return type == RTE_TYPE_BF16 || type == RTE_TYPE_F16 || type == RTE_TYPE_F32; }

}  // namespace

#define ST(s) static_cast<cudaStream_t>(s)
#define BY_TYPE(type, CALL)                             \
  do {                                                  \
    if (type == RTE_TYPE_BF16) CALL(__nv_bfloat16);     \
    else if (type == RTE_TYPE_F16) CALL(__half);        \
    else CALL(float);                                   \
  } while (0)

extern "C" int rte_token_logprobs_fwd(const void* logits, int32_t type, int64_t ldl, const int64_t* tokens, int64_t ignore_index, float temperature, int32_t top_k,
                                      float* logprob, float* entropy, float* top_logprobs, int64_t* top_ids, float* row_stats, int32_t rows, int32_t V, int32_t* status,
                                      rte_stream_t stream) {
  RTE_CHECK_ARG(logits && tokens && logprob && entropy && row_stats && type_ok(type) && rows > 0 && V > 0 && ldl >= 0 && temperature_ok(temperature));
  RTE_CHECK_ARG(top_k >= 0 && top_k <= V && top_k <= TS_MAX_LIST && (top_k == 0 || (top_logprobs && top_ids)));
#define CALL(T)                                                                                                                                                     \
  rte::launch(token_logprobs_kernel<T>, rows, TS_THREADS, 0, ST(stream), static_cast<const T*>(logits), ldl, tokens, ignore_index, 1.f / temperature, top_k, logprob, \
              entropy, top_logprobs, top_ids, reinterpret_cast<float2*>(row_stats), V, status)
  BY_TYPE(type, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}

extern "C" int rte_token_logprobs_bwd(const void* logits, int32_t type, int64_t ldl, const int64_t* tokens, float temperature, int32_t top_k, const int64_t* top_ids,
                                      const float* row_stats, const float* entropy, const float* g_logprob, const float* g_entropy, const float* g_top, void* dlogits,
                                      int32_t rows, int32_t V, rte_stream_t stream) {
  RTE_CHECK_ARG(logits && tokens && entropy && row_stats && dlogits && type_ok(type) && rows > 0 && V > 0 && ldl >= 0 && temperature_ok(temperature));
  RTE_CHECK_ARG(top_k >= 0 && top_k <= V && top_k <= TS_MAX_LIST && (!g_top || top_k == 0 || top_ids));
#define CALL(T)                                                                                                                                                      \
  rte::launch(token_logprobs_bwd_kernel<T>, rows, TS_THREADS, 0, ST(stream), static_cast<const T*>(logits), ldl, tokens, 1.f / temperature, top_k, top_ids,           \
              reinterpret_cast<const float2*>(row_stats), entropy, g_logprob, g_entropy, g_top, static_cast<T*>(dlogits), V)
  BY_TYPE(type, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}

extern "C" int rte_distill_topk_fwd(const void* logits, int32_t type, int64_t ldl, const float* teacher, const int64_t* ids, int32_t k, float temperature, int32_t tail,
                                    float* loss, float* row_stats, int32_t rows, int32_t V, int32_t* status, rte_stream_t stream) {
  RTE_CHECK_ARG(logits && teacher && ids && loss && row_stats && type_ok(type) && rows > 0 && V > 0 && ldl >= 0 && temperature_ok(temperature));
  RTE_CHECK_ARG(k > 0 && k <= TS_MAX_LIST);
  if (reinterpret_cast<uintptr_t>(row_stats) & 15) return RTE_ERR_ALIGNMENT;
#define CALL(T)                                                                                                                                                     \
  rte::launch(distill_topk_kernel<T>, rows, TS_THREADS, 0, ST(stream), static_cast<const T*>(logits), ldl, teacher, ids, k, temperature, tail, loss,                  \
              reinterpret_cast<float4*>(row_stats), V, status)
  BY_TYPE(type, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}

extern "C" int rte_distill_topk_bwd(const void* logits, int32_t type, int64_t ldl, const float* teacher, const int64_t* ids, int32_t k, float temperature,
                                    const float* row_stats, const float* dloss, void* dlogits, int32_t rows, int32_t V, rte_stream_t stream) {
  RTE_CHECK_ARG(logits && teacher && ids && row_stats && dloss && dlogits && type_ok(type) && rows > 0 && V > 0 && ldl >= 0 && temperature_ok(temperature));
  RTE_CHECK_ARG(k > 0 && k <= TS_MAX_LIST);
  if (reinterpret_cast<uintptr_t>(row_stats) & 15) return RTE_ERR_ALIGNMENT;
#define CALL(T)                                                                                                                                                 \
  rte::launch(distill_topk_bwd_kernel<T>, rows, TS_THREADS, 0, ST(stream), static_cast<const T*>(logits), ldl, teacher, ids, k, temperature,                      \
              reinterpret_cast<const float4*>(row_stats), dloss, static_cast<T*>(dlogits), V)
  BY_TYPE(type, CALL);
#undef CALL
  RTE_LAUNCH_CHECK();
  return RTE_OK;
}
