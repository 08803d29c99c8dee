// Log-probabilities of item lists under catalogue scores, and the preference loss of pairs of such
// lists (paired log ratios against a reference model), forward and backward (gfx950).
//
// Scores x[s, t, :] of list s at place t, item y[s, t]:
//   lse = log sum_j exp(x_j),   logp[s] = sum_t (x[y] - lse)      (over the places in use; / their number)
//   h_p = beta * ((logp[p] - ref[p]) - (logp[P + p] - ref[P + p]))
//   loss = mean_p  (1 - e) softplus(-h) + e softplus(h)           (hinge and squared forms: pair_term)
//   dx[s, t, j] = c_s * ([j = y] - exp(x_j - lse)),  c_s = dloss/dlogp[s]
//
// The rows are read once forward (maximum and sum of exponentials in one pass, rescaled when the
// maximum grows) and once backward, where every gradient element is written once; the row's maximum
// and log-sum are kept, the probabilities are not.  Places that are not in use are not read at all;
// their gradient is zero.  Long rows are cut into parts so that few rows still fill the GPU; the
// parts' maxima and sums are joined in order.  All statistics and sums are fp32 or wider.
#include <algorithm>

#include "elem.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / rk::kWave;

struct Rows {
  int64_t stride_s, stride_t;   // of the scores, in elements
  int32_t S, T, V;              // lists, places, catalogue
  int32_t parts, part_len;      // every row is cut into `parts` parts of part_len scores
  const int64_t *items;         // [S, T]
  int64_t ld_items;
  int64_t ignore;
};

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// (max, sum) pairs: sum counts exp(x - max).  The maximum starts at the lowest finite float, so that a
// row of nothing but -inf gives sum 0 and a log of -inf, not a NaN from inf - inf.
__device__ __forceinline__ void merge(float &m, float &s, float om, float os) {
  const float nm = fmaxf(m, om);
  s = s * __expf(m - nm) + os * __expf(om - nm);
  m = nm;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void rows_fwd_kernel(Rows a, const T *__restrict__ x, float2 *__restrict__ part,
                                                            int32_t *__restrict__ ticket) {
  constexpr int VEC = rk::Elem<T>::kVec, U = 4;
  __shared__ float s_m[kWaves], s_s[kWaves];
  if (blockIdx.x == 0 && threadIdx.x == 0) ticket[0] = 0;   // for the closing launch
  const int64_t row = blockIdx.x / a.parts;
  const int32_t p = (int32_t)(blockIdx.x - row * a.parts), s = (int32_t)(row / a.T), t = (int32_t)(row - (int64_t)s * a.T);
  if (a.items[s * a.ld_items + t] == a.ignore) return;
  const int32_t lo = p * a.part_len, hi = min(a.V, lo + a.part_len);
  const T *r = x + s * a.stride_s + t * a.stride_t;
  float m = -__FLT_MAX__, sum = 0.0f;
  int32_t j = lo + (int32_t)threadIdx.x * VEC;
  for (; j + (U - 1) * kThreads * VEC + VEC <= hi; j += U * kThreads * VEC) {
    rk::Pack<T, VEC> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].load(r + j + u * kThreads * VEC);
    float f[U][VEC], top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u].widen(f[u]);
#pragma unroll
      for (int e = 0; e < VEC; ++e) top = fmaxf(top, f[u][e]);
    }
    sum *= __expf(m - top);
    m = top;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum += __expf(f[u][e] - m);
  }
  for (; j < hi; j += kThreads * VEC) {
    float f[VEC], top = m;
    if (j + VEC <= hi) {
      rk::Pack<T, VEC> v;
      v.load(r + j);
      v.widen(f);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = j + e < hi ? rk::Elem<T>::get(r[j + e]) : neg_inf();
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) top = fmaxf(top, f[e]);
    sum *= __expf(m - top);
    m = top;
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum += __expf(f[e] - m);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float om = __shfl_xor(m, off, rk::kWave), os = __shfl_xor(sum, off, rk::kWave);
    merge(m, sum, om, os);
  }
  if (threadIdx.x % rk::kWave == 0) {
    s_m[threadIdx.x / rk::kWave] = m;
    s_s[threadIdx.x / rk::kWave] = sum;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) merge(m, sum, s_m[w], s_s[w]);
    part[blockIdx.x] = make_float2(m, sum);
  }
}

// one wavefront: the log-probability of list s; leaves (max, log sum) of its rows in stat
template <typename T>
__device__ __forceinline__ float list_logp(const Rows &a, const T *__restrict__ x, const float2 *__restrict__ part,
                                           float2 *__restrict__ stat, int32_t s, int average, int32_t &used) {
  const int lane = threadIdx.x % rk::kWave;
  double sum = 0.0;
  int32_t n = 0;
  for (int32_t t = lane; t < a.T; t += rk::kWave) {
    const int64_t y = a.items[s * a.ld_items + t], row = (int64_t)s * a.T + t;
    if (y == a.ignore) continue;
    float m = -__FLT_MAX__, q = 0.0f;
    for (int p = 0; p < a.parts; ++p) {
      const float2 o = part[row * a.parts + p];
      merge(m, q, o.x, o.y);
    }
    const float lq = logf(q);
    stat[row] = make_float2(m, lq);
    // an item outside the catalogue has no score: its log-probability is not a number
    const float xy = y >= 0 && y < a.V ? rk::Elem<T>::get(x[s * a.stride_s + t * a.stride_t + y]) : __builtin_nanf("");
    sum += (double)((xy - m) - lq);
    ++n;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    sum += __shfl_xor(sum, off, rk::kWave);
    n += __shfl_xor(n, off, rk::kWave);
  }
  used = n;
  return (float)(average && n > 0 ? sum / n : sum);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void lists_kernel(Rows a, const T *__restrict__ x, const float2 *__restrict__ part,
                                                         float2 *__restrict__ stat, int average, float *__restrict__ logps,
                                                         int32_t *__restrict__ used) {
  const int32_t s = (int32_t)blockIdx.x * kWaves + threadIdx.x / rk::kWave;
  if (s >= a.S) return;
  int32_t n;
  const float v = list_logp(a, x, part, stat, s, average, n);
  if (threadIdx.x % rk::kWave == 0) {
    logps[s] = v;
    used[s] = n;
  }
}

__device__ __forceinline__ float softplus(float z) { return fmaxf(z, 0.0f) + log1pf(expf(-fabsf(z))); }
__device__ __forceinline__ float sigmoid(float z) {
  const float e = expf(-fabsf(z));
  return (z >= 0.0f ? 1.0f : e) / (1.0f + e);
}

// the term of one pair and its derivative by (log ratio of the preferred - log ratio of the other)
__device__ __forceinline__ float pair_term(float d, float beta, float eps, int kind, float &slope) {
  if (kind == RK_PREF_SQUARED) {
    const float e = d - 0.5f / beta;
    slope = 2.0f * e;
    return e * e;
  }
  const float h = beta * d;
  if (kind == RK_PREF_HINGE) {
    const float e = 1.0f - h;
    slope = e > 0.0f ? -beta : (e <= 0.0f ? 0.0f : e);   // (NaN stays NaN)
    return e > 0.0f ? e : (e <= 0.0f ? 0.0f : e);
  }
  slope = beta * (eps * sigmoid(h) - (1.0f - eps) * sigmoid(-h));
  // (a smoothing of 0 or 1 leaves one of the terms out: 0 * inf is not a number)
  float term = eps < 1.0f ? (1.0f - eps) * softplus(-h) : 0.0f;
  if (eps > 0.0f) term += eps * softplus(h);
  return term;
}

// Pairs p and P + p, one wavefront each; the workgroup that finishes last adds the pairs' terms in
// order.  Every pair's term reaches memory by an agent-scope store in front of its ticket and is read
// back by an agent-scope load behind the last ticket: the workgroups run under different L2 caches.
template <typename T>
__global__ __launch_bounds__(kThreads) void pairs_kernel(Rows a, const T *__restrict__ x, const float2 *__restrict__ part,
                                                         float2 *__restrict__ stat, const float *__restrict__ ref,
                                                         int average, float beta, float eps, int kind,
                                                         float *__restrict__ logps, int32_t *__restrict__ used,
                                                         float *__restrict__ slope_out, float *__restrict__ terms,
                                                         int32_t *__restrict__ ticket, float *__restrict__ loss) {
  __shared__ int s_last;
  __shared__ double s_sum[kWaves];
  const int lane = threadIdx.x % rk::kWave;
  const int32_t P = a.S / 2, p = (int32_t)blockIdx.x * kWaves + threadIdx.x / rk::kWave;
  if (p < P) {
    int32_t nc, nr;
    const float c = list_logp(a, x, part, stat, p, average, nc);
    const float r = list_logp(a, x, part, stat, P + p, average, nr);
    if (lane == 0) {
      float slope;
      const float term = pair_term((c - ref[p]) - (r - ref[P + p]), beta, eps, kind, slope);
      logps[p] = c;
      logps[P + p] = r;
      used[p] = nc;
      used[P + p] = nr;
      slope_out[p] = slope / (float)P;
      slope_out[P + p] = -slope / (float)P;
      __hip_atomic_store(&terms[p], term, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0)
    s_last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int32_t)gridDim.x - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double sum = 0.0;
  for (int32_t i = threadIdx.x; i < P; i += kThreads)
    sum += (double)__hip_atomic_load(&terms[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, rk::kWave);
  if (lane == 0) s_sum[threadIdx.x / rk::kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = s_sum[0];
    for (int w = 1; w < kWaves; ++w) all += s_sum[w];
    loss[0] = (float)(all / P);
  }
}

// dx = c * ([j = y] - exp((x - max) - log sum)), c = (g_loss * slope + g_logps) of the row's list
template <typename T>
__global__ __launch_bounds__(kThreads) void rows_bwd_kernel(Rows a, const T *__restrict__ x, const float2 *__restrict__ stat,
                                                            const float *__restrict__ g_loss, const float *__restrict__ slope,
                                                            const float *__restrict__ g_logps, int average,
                                                            const int32_t *__restrict__ used, T *__restrict__ dx) {
  constexpr int VEC = rk::Elem<T>::kVec, U = 4;
  const int64_t row = blockIdx.x / a.parts;
  const int32_t p = (int32_t)(blockIdx.x - row * a.parts), s = (int32_t)(row / a.T), t = (int32_t)(row - (int64_t)s * a.T);
  const int32_t lo = p * a.part_len, hi = min(a.V, lo + a.part_len);
  const int64_t y = a.items[s * a.ld_items + t];
  T *d = dx + row * a.V;
  if (y == a.ignore) {
    rk::Pack<T, VEC> zero;
#pragma unroll
    for (int i = 0; i < rk::Pack<T, VEC>::kWords; ++i) zero.w[i] = 0u;
    for (int32_t j = lo + (int32_t)threadIdx.x * VEC; j < hi; j += kThreads * VEC) {
      if (j + VEC <= hi) {
        zero.store(d + j);
      } else {
        for (int e = 0; e < VEC && j + e < hi; ++e) d[j + e] = rk::Elem<T>::put(0.0f);
      }
    }
    return;
  }
  const T *r = x + s * a.stride_s + t * a.stride_t;
  float c = (g_loss ? g_loss[0] * slope[s] : 0.0f) + (g_logps ? g_logps[s] : 0.0f);
  if (average) c /= (float)used[s];
  const float2 st = stat[row];
  const int32_t label = y >= 0 && y < a.V ? (int32_t)y : -1;
  if (label < 0) c = __builtin_nanf("");
  auto one = [&](const rk::Pack<T, VEC> &v, int32_t j) {
    float f[VEC];
    v.widen(f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = -c * __expf((f[e] - st.x) - st.y);
    if ((uint32_t)(label - j) < (uint32_t)VEC) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (label - j == e) f[e] += c;
    }
    rk::Pack<T, VEC> o;
    o.narrow(f);
    o.store(d + j);
  };
  int32_t j = lo + (int32_t)threadIdx.x * VEC;
  for (; j + (U - 1) * kThreads * VEC + VEC <= hi; j += U * kThreads * VEC) {
    rk::Pack<T, VEC> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].load(r + j + u * kThreads * VEC);
#pragma unroll
    for (int u = 0; u < U; ++u) one(v[u], j + u * kThreads * VEC);
  }
  for (; j < hi; j += kThreads * VEC) {
    if (j + VEC <= hi) {
      rk::Pack<T, VEC> v;
      v.load(r + j);
      one(v, j);
    } else {
      for (int e = 0; e < VEC && j + e < hi; ++e) {
        float f = -c * __expf((rk::Elem<T>::get(r[j + e]) - st.x) - st.y);
        if (label == j + e) f += c;
        d[j + e] = rk::Elem<T>::put(f);
      }
    }
  }
}

// parts of a row: enough workgroups for the GPU, parts of at least kMinPart scores
constexpr int kMinPart = 4096, kWantBlocks = 2048;
void cut(Rows &a) {
  const int64_t rows = (int64_t)a.S * a.T;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(rk::ceil_div(kWantBlocks, rows), rk::ceil_div(a.V, kMinPart)));
  a.part_len = (int32_t)(rk::ceil_div(rk::ceil_div(a.V, want), 8) * 8);
  a.parts = (int32_t)rk::ceil_div(a.V, a.part_len);
}

int make_rows(Rows &a, int32_t dtype, int32_t S, int32_t T, int32_t V, int64_t stride_s, int64_t stride_t,
              const int64_t *items, int64_t ld_items, int64_t ignore) {
  RK_CHECK_ARG(dtype == RK_F32 || dtype == RK_BF16 || dtype == RK_F16, "unknown element type %d", dtype);
  RK_CHECK_ARG(S >= 0 && T >= 0 && V >= 1, "bad size: %d lists, %d places, %d items", S, T, V);
  // a part's last step may look a few thousand scores past its end before it stops
  RK_CHECK_ARG(V < (1 << 30), "more than 2^30 items");
  a = {stride_s, stride_t, S, T, V, 0, 0, items, ld_items, ignore};
  if (S == 0 || T == 0) return RK_OK;
  RK_CHECK_ARG(items, "null pointer");
  cut(a);
  RK_CHECK_ARG((int64_t)S * T * a.parts < INT32_MAX, "too many rows");
  return RK_OK;
}

struct Ws {   // of the forward calls, in 4-byte words: parts' (max, sum), pairs' terms, ticket
  int64_t part, terms, ticket, words;
};
Ws ws_of(const Rows &a) {
  Ws w;
  w.part = 0;
  w.terms = 2 * (int64_t)a.S * a.T * a.parts;
  w.ticket = w.terms + a.S;
  w.words = w.ticket + 4;
  return w;
}

template <typename T>
int launch_rows_fwd(const Rows &a, const void *x, float *ws, const Ws &w, hipStream_t st) {
  rows_fwd_kernel<T><<<(uint32_t)((int64_t)a.S * a.T * a.parts), kThreads, 0, st>>>(
      a, (const T *)x, (float2 *)(ws + w.part), (int32_t *)(ws + w.ticket));
  RK_CHECK_LAUNCH("rows_fwd_kernel");
  return RK_OK;
}

template <typename T>
int run_lists(const Rows &a, const void *x, int average, float *stat, float *logps, int32_t *used, float *ws,
              hipStream_t st) {
  const Ws w = ws_of(a);
  if (int rc = launch_rows_fwd<T>(a, x, ws, w, st)) return rc;
  lists_kernel<T><<<(uint32_t)rk::ceil_div(a.S, kWaves), kThreads, 0, st>>>(a, (const T *)x, (const float2 *)(ws + w.part),
                                                                          (float2 *)stat, average, logps, used);
  RK_CHECK_LAUNCH("lists_kernel");
  return RK_OK;
}

template <typename T>
int run_pairs(const Rows &a, const void *x, const float *ref, int average, float beta, float eps, int kind, float *stat,
              float *logps, int32_t *used, float *slope, float *loss, float *ws, hipStream_t st) {
  const Ws w = ws_of(a);
  if (int rc = launch_rows_fwd<T>(a, x, ws, w, st)) return rc;
  pairs_kernel<T><<<(uint32_t)rk::ceil_div(a.S / 2, kWaves), kThreads, 0, st>>>(
      a, (const T *)x, (const float2 *)(ws + w.part), (float2 *)stat, ref, average, beta, eps, kind, logps, used, slope,
      ws + w.terms, (int32_t *)(ws + w.ticket), loss);
  RK_CHECK_LAUNCH("pairs_kernel");
  return RK_OK;
}

template <typename T>
int run_bwd(const Rows &a, const void *x, const float *stat, const float *g_loss, const float *slope, const float *g_logps,
            int average, const int32_t *used, void *dx, hipStream_t st) {
  rows_bwd_kernel<T><<<(uint32_t)((int64_t)a.S * a.T * a.parts), kThreads, 0, st>>>(
      a, (const T *)x, (const float2 *)stat, g_loss, slope, g_logps, average, used, (T *)dx);
  RK_CHECK_LAUNCH("rows_bwd_kernel");
  return RK_OK;
}

}  // namespace

extern "C" {

size_t rk_list_logps_ws_bytes(int32_t S, int32_t T, int32_t V) {
  if (S <= 0 || T <= 0 || V <= 0) return 0;
  Rows a = {0, 0, S, T, V, 0, 0, nullptr, 0, 0};
  cut(a);
  return (size_t)ws_of(a).words * 4;
}

#define RK_BY_TYPE(fn, ...)                               \
  (dtype == RK_F32 ? fn<float>(__VA_ARGS__)               \
                   : dtype == RK_BF16 ? fn<__bf16>(__VA_ARGS__) : fn<_Float16>(__VA_ARGS__))

int rk_list_logps_fwd(const void *scores, int32_t dtype, int32_t S, int32_t T, int32_t V, int64_t stride_s,
                      int64_t stride_t, const int64_t *items, int64_t ld_items, int64_t ignore_index, int32_t average,
                      float *stat, float *logps, int32_t *used, void *ws, size_t ws_bytes, void *stream) {
  Rows a;
  if (int rc = make_rows(a, dtype, S, T, V, stride_s, stride_t, items, ld_items, ignore_index)) return rc;
  RK_CHECK_ARG(S == 0 || T > 0, "lists without places");
  if (S == 0) return RK_OK;
  RK_CHECK_ARG(scores && stat && logps && used && ws, "null pointer");
  RK_CHECK_ARG(ws_bytes >= rk_list_logps_ws_bytes(S, T, V), "workspace too small");
  return RK_BY_TYPE(run_lists, a, scores, average, stat, logps, used, (float *)ws, (hipStream_t)stream);
}

int rk_preference_fwd(const void *scores, int32_t dtype, int32_t S, int32_t T, int32_t V, int64_t stride_s,
                      int64_t stride_t, const int64_t *items, int64_t ld_items, int64_t ignore_index, int32_t average,
                      const float *ref_logps, float beta, float label_smoothing, int32_t kind, float *stat, float *logps,
                      int32_t *used, float *slope, float *loss, void *ws, size_t ws_bytes, void *stream) {
  Rows a;
  if (int rc = make_rows(a, dtype, S, T, V, stride_s, stride_t, items, ld_items, ignore_index)) return rc;
  RK_CHECK_ARG(S >= 2 && S % 2 == 0 && T > 0, "pairs of lists are needed: %d lists of %d places", S, T);
  RK_CHECK_ARG(kind == RK_PREF_SIGMOID || kind == RK_PREF_HINGE || kind == RK_PREF_SQUARED, "unknown kind %d", kind);
  RK_CHECK_ARG(beta > 0.0f, "beta must be positive");
  RK_CHECK_ARG(label_smoothing >= 0.0f && label_smoothing <= 1.0f, "label smoothing outside [0, 1]");
  RK_CHECK_ARG(label_smoothing == 0.0f || kind == RK_PREF_SIGMOID, "label smoothing is part of the sigmoid form only");
  RK_CHECK_ARG(scores && ref_logps && stat && logps && used && slope && loss && ws, "null pointer");
  RK_CHECK_ARG(ws_bytes >= rk_list_logps_ws_bytes(S, T, V), "workspace too small");
  return RK_BY_TYPE(run_pairs, a, scores, ref_logps, average, beta, label_smoothing, kind, stat, logps, used, slope, loss,
                    (float *)ws, (hipStream_t)stream);
}

int rk_list_logps_bwd(const void *scores, int32_t dtype, int32_t S, int32_t T, int32_t V, int64_t stride_s,
                      int64_t stride_t, const int64_t *items, int64_t ld_items, int64_t ignore_index, int32_t average,
                      const float *stat, const int32_t *used, const float *g_loss, const float *slope,
                      const float *g_logps, void *d_scores, void *stream) {
  Rows a;
  if (int rc = make_rows(a, dtype, S, T, V, stride_s, stride_t, items, ld_items, ignore_index)) return rc;
  if (S == 0 || T == 0) return RK_OK;
  RK_CHECK_ARG(scores && stat && used && d_scores, "null pointer");
  RK_CHECK_ARG(!g_loss || slope, "the gradient of the loss needs the slopes of rk_preference_fwd");
  return RK_BY_TYPE(run_bwd, a, scores, stat, g_loss, slope, g_logps, average, used, d_scores, (hipStream_t)stream);
}

}  // extern "C"
