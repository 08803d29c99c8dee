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
constexpr int kPairThreads = 1024;
// Rows that one workgroup joins, in the launch of the pairs: one launch fewer, which a call from the host notices (a step
// over 4000 rows of 300 scores: 53 us, with two launches 57) and a recorded one does not (forward 13.5 us, 9.8).
constexpr int kFewRows = 4096;
// Pairs that one workgroup adds up behind more rows than that; more take two launches (4096 pairs 7.2 us, in two
// launches 2.9 + 1.8 and a gap; 100000 pairs 129 us, 4.9 + 4.7).
constexpr int kOnePairs = 4096;
constexpr int kLongList = 512;       // places of a list that a wavefront adds up

// A row's part is read by a workgroup, or by a wavefront (four parts in a workgroup): a row of 1000 scores
// keeps 125 of 256 threads busy once.
struct Rows {
  int64_t stride_s, stride_t;   // of the scores, in elements
  int32_t S, T, V;              // lists, places, catalogue
  int32_t parts, part_len;      // every row is cut into `parts` parts of part_len scores
  const int64_t *items;         // [S, T]
  int64_t ld_items;
  int64_t ignore;
  uint32_t units;               // S * T * parts, below 2^31
};

// which (row, part) a thread works on: the grid has two dimensions because one ends at 2^32 threads
template <int TPR>
__device__ __forceinline__ uint32_t unit_index() {   // (units < 2^31; the same for a wavefront, kept in scalar registers)
  const uint32_t block = blockIdx.y * gridDim.x + blockIdx.x;
  return TPR == kThreads ? block : __builtin_amdgcn_readfirstlane(block * (kThreads / TPR) + threadIdx.x / TPR);
}

__device__ __forceinline__ float neg_inf() { return -__builtin_inff(); }

// (max, sum) pairs: sum counts exp(x - max).  The maximum starts at the lowest finite float, so that a
// row of nothing but -inf gives sum 0 and a log of -inf, not a NaN from inf - inf.
__device__ __forceinline__ void merge(float &m, float &s, float om, float os) {
  const float nm = fmaxf(m, om);
  s = s * __expf(m - nm) + os * __expf(om - nm);
  m = nm;
}

// One part of one row: its (max, sum) and, if the row's item lies in it, the item's score.  The next step's
// vectors are on their way while a step's exponentials are computed.
template <typename T, int TPR>   // TPR: threads of a part, 256 or 64
__global__ __launch_bounds__(kThreads) void rows_fwd_kernel(Rows a, const T *__restrict__ x, float2 *__restrict__ part,
                                                            float *__restrict__ score) {
  constexpr int VEC = rk::Elem<T>::kVec, U = 4, kStep = U * TPR * VEC;
  __shared__ float s_m[kWaves], s_s[kWaves];
  const uint32_t unit = unit_index<TPR>();
  if (unit >= a.units) return;
  const int lane = TPR == kThreads ? threadIdx.x : threadIdx.x % TPR;
  const uint32_t row = unit / (uint32_t)a.parts;
  const int32_t p = (int32_t)(unit - row * a.parts), s = (int32_t)(row / (uint32_t)a.T), t = (int32_t)(row - (uint32_t)s * a.T);
  const int64_t y = a.items[s * a.ld_items + t];
  if (y == a.ignore) return;
  const int32_t lo = p * a.part_len, hi = min(a.V, lo + a.part_len);
  const T *r = x + s * a.stride_s + t * a.stride_t;
  if (lane == 0) {
    if (y >= lo && y < hi)
      score[row] = rk::Elem<T>::get(r[y]);
    else if (p == 0 && (y < 0 || y >= a.V))
      score[row] = __builtin_nanf("");   // an item outside the catalogue has no score
  }
  float m = -__FLT_MAX__, sum = 0.0f;
  auto add = [&](const float *f, int n) {
    float top = m;
    for (int e = 0; e < n; ++e) top = fmaxf(top, f[e]);
    sum *= __expf(m - top);
    m = top;
    for (int e = 0; e < n; ++e) sum += __expf(f[e] - m);
  };
  const int32_t steps = (hi - lo) / kStep;
  const T *q = r + lo + lane * VEC;
  rk::Pack<T, VEC> v[U];
  if (steps > 0)
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].load(q + u * TPR * VEC);
  for (int32_t k = 0; k < steps; ++k) {
    float f[U * VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].widen(*reinterpret_cast<float(*)[VEC]>(f + u * VEC));
    q += kStep;
    if (k + 1 < steps)
#pragma unroll
      for (int u = 0; u < U; ++u) v[u].load(q + u * TPR * VEC);
    add(f, U * VEC);
  }
  // the rest of the part: less than one step
  int32_t j = lo + steps * kStep + lane * VEC;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (j + u * TPR * VEC + VEC <= hi) v[u].load(r + j + u * TPR * VEC);
#pragma unroll
  for (int u = 0; u < U; ++u, j += TPR * VEC) {
    float f[VEC];
    if (j + VEC <= hi) {
      v[u].widen(f);
      add(f, VEC);
    } else if (j < hi) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = j + e < hi ? rk::Elem<T>::get(r[j + e]) : neg_inf();
      add(f, VEC);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const float om = __shfl_xor(m, off, rk::kWave), os = __shfl_xor(sum, off, rk::kWave);
    merge(m, sum, om, os);
  }
  if constexpr (TPR == rk::kWave) {
    if (lane == 0) part[unit] = make_float2(m, sum);
    return;
  }
  if (threadIdx.x % rk::kWave == 0) {
    s_m[threadIdx.x / rk::kWave] = m;
    s_s[threadIdx.x / rk::kWave] = sum;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) merge(m, sum, s_m[w], s_s[w]);
    part[unit] = make_float2(m, sum);
  }
}

// log-probability of the row's item from the row's parts, which it joins in order; leaves (max, log sum)
__device__ __forceinline__ float row_logp(const Rows &a, int64_t row, const float2 *__restrict__ part,
                                          const float *__restrict__ score, float2 *__restrict__ stat) {
  float m = -__FLT_MAX__, q = 0.0f;
#pragma unroll 4
  for (int p = 0; p < a.parts; ++p) {
    const float2 o = part[row * a.parts + p];
    merge(m, q, o.x, o.y);
  }
  const float lq = logf(q);
  stat[row] = make_float2(m, lq);
  return (score[row] - m) - lq;
}

// The lists' log-probabilities and the numbers of their places in use.  `lanes` threads for a list: a power of two up
// to 64 (200000 lists of one place: 5.1 us, by a wavefront each 51), or 1024 where a list is long (LONG; two lists
// of 100000 places: 104 us, by a wavefront each 1340; eight of 600: 4.0 and 10.7).
template <bool LONG>
__global__ __launch_bounds__(LONG ? kPairThreads : kThreads) void lists_kernel(Rows a, const float2 *__restrict__ part,
                                                                              const float *__restrict__ score,
                                                                              float2 *__restrict__ stat, int average, int lanes,
                                                                              float *__restrict__ logps,
                                                                              int32_t *__restrict__ used) {
  const int64_t s = LONG ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * kThreads + threadIdx.x) / lanes;
  const int lane = (int)threadIdx.x & (lanes - 1);
  if (s >= a.S) return;
  double sum = 0.0;
  int32_t n = 0;
  for (int32_t t = lane; t < a.T; t += lanes) {
    if (a.items[s * a.ld_items + t] == a.ignore) continue;
    sum += (double)row_logp(a, s * a.T + t, part, score, stat);
    ++n;
  }
  for (int off = min(lanes, rk::kWave) / 2; off > 0; off >>= 1) {
    sum += __shfl_xor(sum, off, rk::kWave);
    n += __shfl_xor(n, off, rk::kWave);
  }
  if constexpr (LONG) {
    __shared__ double s_sum[kPairThreads / rk::kWave];
    __shared__ int32_t s_n[kPairThreads / rk::kWave];
    if (threadIdx.x % rk::kWave == 0) {
      s_sum[threadIdx.x / rk::kWave] = sum;
      s_n[threadIdx.x / rk::kWave] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0)
      for (int w = 1; w < kPairThreads / rk::kWave; ++w) {
        sum += s_sum[w];
        n += s_n[w];
      }
  }
  if (lane == 0) {
    logps[s] = (float)(average && n > 0 ? sum / n : sum);
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

// One workgroup: the pairs' terms, their slopes and the mean, added in a fixed order.  K > 0: it also forms the
// lists' log-probabilities, from up to K rows for each thread (one launch instead of two), or a row for each `lanes`
// threads, a power of two (two rows of 10^8 scores, 4096 parts each: 15 us where a thread for each took 494).
template <int K>
__global__ __launch_bounds__(kPairThreads) void pairs_kernel(Rows a, const float2 *__restrict__ part,
                                                             const float *__restrict__ score, float2 *__restrict__ stat,
                                                             const float *__restrict__ ref, int average, float beta,
                                                             float eps, int kind, int lanes, float *__restrict__ logps,
                                                             int32_t *__restrict__ used, float *__restrict__ slope_out,
                                                             float *__restrict__ loss) {
  constexpr bool ROWS = K > 0;
  __shared__ float s_row[ROWS ? K * kPairThreads : 1], s_logp[ROWS ? K * kPairThreads : 1];
  __shared__ double s_sum[kPairThreads / rk::kWave];
  const int32_t P = a.S / 2;
  if constexpr (ROWS) {
    const int32_t rows = a.S * a.T;
    const int32_t sub = (int32_t)threadIdx.x & (lanes - 1);
    bool in[K];                                            // (the loads of a thread's rows are in flight together)
    int32_t at[K];
    float m[K], q[K], sc[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      at[k] = (k * kPairThreads + (int32_t)threadIdx.x) / lanes;
      const int32_t row = min(at[k], rows - 1), s = row / a.T, t = row - s * a.T;
      in[k] = at[k] < rows && a.items[s * a.ld_items + t] != a.ignore;
      sc[k] = score[row];                                  // (not written for a place that is not in use, and not used)
      m[k] = -__FLT_MAX__;
      q[k] = 0.0f;
    }
    constexpr int U = K == 1 ? 8 : 1;                      // parts of a thread in flight
    for (int p = sub; p < a.parts; p += U * lanes) {
      float2 o[U][K];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < K; ++k)
          o[u][k] = part[(int64_t)min(at[k], rows - 1) * a.parts + min(p + u * lanes, a.parts - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (p + u * lanes < a.parts) merge(m[k], q[k], o[u][k].x, o[u][k].y);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      for (int off = lanes / 2; off > 0; off >>= 1) {
        const float om = __shfl_xor(m[k], off, rk::kWave), os = __shfl_xor(q[k], off, rk::kWave);
        merge(m[k], q[k], om, os);
      }
      const int32_t row = at[k];
      if (row >= rows || sub != 0) continue;
      const float lq = logf(q[k]);
      if (in[k]) stat[row] = make_float2(m[k], lq);
      // a place that is not in use is marked by the one value that no log-probability has
      s_row[row] = in[k] ? (sc[k] - m[k]) - lq : __builtin_inff();
    }
    __syncthreads();
    // up to 16 lanes for every list
    const int per_list = a.T >= 16 ? 16 : a.T > 4 ? 8 : a.T > 1 ? 4 : 1, place = threadIdx.x & (per_list - 1);
    for (int32_t s0 = 0; s0 < a.S; s0 += kPairThreads / per_list) {
      const int32_t s = s0 + (int32_t)threadIdx.x / per_list;
      double sum = 0.0;
      int32_t n = 0;
      if (s < a.S)
        for (int32_t t = place; t < a.T; t += per_list) {
          const float v = s_row[s * a.T + t];
          if (v == __builtin_inff()) continue;
          sum += (double)v;
          ++n;
        }
      for (int off = per_list / 2; off > 0; off >>= 1) {
        sum += __shfl_xor(sum, off, rk::kWave);
        n += __shfl_xor(n, off, rk::kWave);
      }
      if (s < a.S && place == 0) {
        const float v = (float)(average && n > 0 ? sum / n : sum);
        s_logp[s] = logps[s] = v;
        used[s] = n;
      }
    }
    __syncthreads();
  }
  double sum = 0.0;
  for (int32_t p = threadIdx.x; p < P; p += kPairThreads) {
    const float c = ROWS ? s_logp[p] : logps[p], r = ROWS ? s_logp[P + p] : logps[P + p];
    float slope;
    sum += (double)pair_term((c - ref[p]) - (r - ref[P + p]), beta, eps, kind, slope);
    slope_out[p] = slope / (float)P;
    slope_out[P + p] = -slope / (float)P;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, rk::kWave);
  if (threadIdx.x % rk::kWave == 0) s_sum[threadIdx.x / rk::kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = s_sum[0];
    for (int w = 1; w < kPairThreads / rk::kWave; ++w) all += s_sum[w];
    loss[0] = (float)(all / P);
  }
}

// Many pairs: their terms and slopes, and one partial sum for every workgroup ...
__global__ __launch_bounds__(kThreads) void terms_kernel(int32_t P, const float *__restrict__ logps, const float *__restrict__ ref,
                                                         float beta, float eps, int kind, float *__restrict__ slope_out,
                                                         double *__restrict__ partial) {
  __shared__ double s_sum[kWaves];
  const int32_t p = (int32_t)blockIdx.x * kThreads + threadIdx.x;
  double sum = 0.0;
  if (p < P) {
    float slope;
    sum = (double)pair_term((logps[p] - ref[p]) - (logps[P + p] - ref[P + p]), beta, eps, kind, slope);
    slope_out[p] = slope / (float)P;
    slope_out[P + p] = -slope / (float)P;
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, rk::kWave);
  if (threadIdx.x % rk::kWave == 0) s_sum[threadIdx.x / rk::kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) partial[blockIdx.x] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

// ... and their mean, by one workgroup.
__global__ __launch_bounds__(kPairThreads) void mean_kernel(int32_t P, const double *__restrict__ partial, int32_t n,
                                                            float *__restrict__ loss) {
  __shared__ double s_sum[kPairThreads / rk::kWave];
  double sum = 0.0;
#pragma unroll 8
  for (int32_t i = threadIdx.x; i < n; i += kPairThreads) sum += partial[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, rk::kWave);
  if (threadIdx.x % rk::kWave == 0) s_sum[threadIdx.x / rk::kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double all = s_sum[0];
    for (int w = 1; w < kPairThreads / rk::kWave; ++w) all += s_sum[w];
    loss[0] = (float)(all / P);
  }
}

// dx = c * ([j = y] - exp((x - max) - log sum)), c = (g_loss * slope + g_logps) of the row's list.  From the
// last row to the first: those were read last and some of them are still cached.  ONCE: a gradient that
// is larger than what the caches should hold is stored past them (left there, its 403 MB were written
// back under the next call's forward launch, which took 74 us instead of 41).
template <typename T, int TPR, bool ONCE>
__global__ __launch_bounds__(kThreads) void rows_bwd_kernel(Rows a, const T *__restrict__ x, const float2 *__restrict__ stat,
                                                            const float *__restrict__ g_loss, const float *__restrict__ slope,
                                                            const float *__restrict__ g_logps, int average,
                                                            const int32_t *__restrict__ used, T *__restrict__ dx) {
  constexpr int VEC = rk::Elem<T>::kVec, U = 4;
  const uint32_t from_end = unit_index<TPR>();
  if (from_end >= a.units) return;
  const uint32_t unit = a.units - 1 - from_end, row = unit / (uint32_t)a.parts;
  const int lane = TPR == kThreads ? threadIdx.x : threadIdx.x % TPR;
  const int32_t p = (int32_t)(unit - row * a.parts), s = (int32_t)(row / (uint32_t)a.T), t = (int32_t)(row - (uint32_t)s * a.T);
  const int32_t lo = p * a.part_len, hi = min(a.V, lo + a.part_len);
  const int64_t y = a.items[s * a.ld_items + t];
  T *d = dx + (int64_t)row * a.V;
  auto put = [&](const rk::Pack<T, VEC> &o, int32_t j) {
    if constexpr (ONCE)
      o.store_once(d + j);
    else
      o.store(d + j);
  };
  if (y == a.ignore) {
    rk::Pack<T, VEC> zero;
#pragma unroll
    for (int i = 0; i < rk::Pack<T, VEC>::kWords; ++i) zero.w[i] = 0u;
    for (int32_t j = lo + lane * VEC; j < hi; j += TPR * VEC) {
      if (j + VEC <= hi) {
        put(zero, j);
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
    put(o, j);
  };
  int32_t j = lo + lane * VEC;
  for (; j + (U - 1) * TPR * VEC + VEC <= hi; j += U * TPR * VEC) {
    rk::Pack<T, VEC> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].load(r + j + u * TPR * VEC);
#pragma unroll
    for (int u = 0; u < U; ++u) one(v[u], j + u * TPR * VEC);
  }
  for (; j < hi; j += TPR * VEC) {
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

// Parts of a row, of at least kMinPart scores: enough workgroups for the GPU, and short ones, whose ends
// do not leave CUs idle (3200 rows of 63001 scores in bf16, 1600 of them in use: forward 41 us with
// 2048 workgroups wanted, 35 with 8192, above that the joining of the parts takes what it gains;
// backward 119 us with 4096, 95 with 32768, 84 with 65536, 89 with parts of 2048).
constexpr int kMinPart = 4096, kWantFwd = 8192, kWantBwd = 65536;
void cut(Rows &a, int want_blocks) {
  const int64_t rows = (int64_t)a.S * a.T;
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>(rk::ceil_div(want_blocks, rows), rk::ceil_div(a.V, kMinPart)));
  a.part_len = (int32_t)(rk::ceil_div(rk::ceil_div(a.V, want), 8) * 8);
  a.parts = (int32_t)rk::ceil_div(a.V, a.part_len);
  a.units = (uint32_t)std::min<int64_t>(rows * a.parts, INT32_MAX);
}

// Up to this many scores a wavefront takes a part.  Microseconds for bf16 rows, by a wavefront / by a workgroup:
// forward 94 / 294 (200000 rows of 100 scores), 47 / 126 (100000 of 1000), 38 / 52 (30000 of 4000), 6.0 / 7.2
// (2000 of 4000); backward 73 / 186, 61 / 96, 4.5 / 5.2 (2000 of 1000), 7.1 / 5.8 (2000 of 2000).
constexpr int kWaveFwd = 4096, kWaveBwd = 1024;
// (few parts: the longer ones by a workgroup.  Whole forward calls over rows of 4096 scores, by a workgroup / by a wavefront:
// 7.4 / 7.6 us for 2 rows, 7.7 / 8.3 for 16, 8.4 / 8.7 for 400, 9.9 / 9.6 for 1000, 12.8 / 11.5 for 2000)
bool fwd_by_wave(const Rows &a) { return a.part_len <= (a.units >= 1024 ? kWaveFwd : kWaveFwd / 2); }

dim3 grid_of(const Rows &a, bool by_wave) {
  const int64_t blocks = rk::ceil_div((int64_t)a.units, by_wave ? kWaves : 1), x = std::min<int64_t>(blocks, 1 << 22);
  return dim3((uint32_t)x, (uint32_t)rk::ceil_div(blocks, x));
}

int make_rows(Rows &a, int32_t dtype, int32_t S, int32_t T, int32_t V, int64_t stride_s, int64_t stride_t,
              const int64_t *items, int64_t ld_items, int64_t ignore, int want_blocks) {
  RK_CHECK_ARG(dtype == RK_F32 || dtype == RK_BF16 || dtype == RK_F16, "unknown element type %d", dtype);
  RK_CHECK_ARG(S >= 0 && T >= 0 && V >= 1, "bad size: %d lists, %d places, %d items", S, T, V);
  // a part's last step may look a few thousand scores past its end before it stops
  RK_CHECK_ARG(V < (1 << 30), "more than 2^30 items");
  a = {stride_s, stride_t, S, T, V, 0, 0, items, ld_items, ignore, 0};
  if (S == 0 || T == 0) return RK_OK;
  RK_CHECK_ARG(items, "null pointer");
  cut(a, want_blocks);
  RK_CHECK_ARG((int64_t)S * T * a.parts < INT32_MAX, "too many rows for one call");
  return RK_OK;
}

struct Ws {   // of the forward calls, in 4-byte words: parts' (max, sum), the items' scores
  int64_t part, score, words;
};
Ws ws_of(const Rows &a) {
  Ws w;
  w.part = 0;
  w.score = 2 * (int64_t)a.S * a.T * a.parts;
  w.words = w.score + (int64_t)a.S * a.T;
  return w;
}

template <typename T>
int launch_rows_fwd(const Rows &a, const void *x, float *ws, const Ws &w, hipStream_t st) {
  if (fwd_by_wave(a))
    rows_fwd_kernel<T, rk::kWave><<<grid_of(a, true), kThreads, 0, st>>>(a, (const T *)x, (float2 *)(ws + w.part), ws + w.score);
  else
    rows_fwd_kernel<T, kThreads><<<grid_of(a, false), kThreads, 0, st>>>(a, (const T *)x, (float2 *)(ws + w.part), ws + w.score);
  RK_CHECK_LAUNCH("rows_fwd_kernel");
  return RK_OK;
}

int launch_lists(const Rows &a, int average, float *stat, float *logps, int32_t *used, const float *ws, const Ws &w,
                 hipStream_t st) {
  if (a.T > kLongList) {
    RK_CHECK_ARG(4 * (int64_t)a.S < rk::kMaxBlocks256, "too many lists for one call");
    lists_kernel<true><<<(uint32_t)a.S, kPairThreads, 0, st>>>(a, (const float2 *)(ws + w.part), ws + w.score, (float2 *)stat,
                                                             average, kPairThreads, logps, used);
    RK_CHECK_LAUNCH("lists_kernel");
    return RK_OK;
  }
  int lanes = 1;
  while (lanes < rk::kWave && lanes < a.T) lanes *= 2;
  const int64_t blocks = rk::ceil_div((int64_t)a.S, kThreads / lanes);
  RK_CHECK_ARG(blocks < rk::kMaxBlocks256, "too many lists for one call");
  lists_kernel<false><<<(uint32_t)blocks, kThreads, 0, st>>>(a, (const float2 *)(ws + w.part), ws + w.score, (float2 *)stat, average,
                                                    lanes, logps, used);
  RK_CHECK_LAUNCH("lists_kernel");
  return RK_OK;
}

template <typename T>
int run_lists(const Rows &a, const void *x, int average, float *stat, float *logps, int32_t *used, float *ws,
              hipStream_t st) {
  const Ws w = ws_of(a);
  if (int rc = launch_rows_fwd<T>(a, x, ws, w, st)) return rc;
  return launch_lists(a, average, stat, logps, used, ws, w, st);
}

template <typename T>
int run_pairs(const Rows &a, const void *x, const float *ref, int average, float beta, float eps, int kind, float *stat,
              float *logps, int32_t *used, float *slope, float *loss, float *ws, hipStream_t st) {
  const Ws w = ws_of(a);
  if (int rc = launch_rows_fwd<T>(a, x, ws, w, st)) return rc;
  const float2 *part = (const float2 *)(ws + w.part);
  const int64_t rows = (int64_t)a.S * a.T;
#define RK_PAIRS(K)                                                                                                    \
  pairs_kernel<K><<<1, kPairThreads, 0, st>>>(a, part, ws + w.score, (float2 *)stat, ref, average, beta, eps, kind, lanes, \
                                              logps, used, slope, loss)
  int lanes = 1;
  if (rows <= kPairThreads) {
    while (lanes < rk::kWave && lanes < a.parts && 2 * lanes * rows <= kPairThreads) lanes *= 2;
    RK_PAIRS(1);
  } else if (rows <= kFewRows) {
    RK_PAIRS(kFewRows / kPairThreads);
  } else {
    if (int rc = launch_lists(a, average, stat, logps, used, ws, w, st)) return rc;
    const int32_t P = a.S / 2, blocks = (int32_t)rk::ceil_div(P, kThreads);
    if (P > kOnePairs) {
      // (the parts are joined: the partial sums take their place)
      terms_kernel<<<blocks, kThreads, 0, st>>>(P, logps, ref, beta, eps, kind, slope, (double *)ws);
      RK_CHECK_LAUNCH("terms_kernel");
      mean_kernel<<<1, kPairThreads, 0, st>>>(P, (const double *)ws, blocks, loss);
      RK_CHECK_LAUNCH("mean_kernel");
      return RK_OK;
    }
    RK_PAIRS(0);
  }
#undef RK_PAIRS
  RK_CHECK_LAUNCH("pairs_kernel");
  return RK_OK;
}

// `stat` and the workspace hold pairs of floats and, behind many rows, doubles
bool aligned8(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

constexpr int64_t kStreamBytes = 64 << 20;   // gradients from this size on are stored past the caches

template <typename T>
int run_bwd(const Rows &a, const void *x, const float *stat, const float *g_loss, const float *slope, const float *g_logps,
            int average, const int32_t *used, void *dx, hipStream_t st) {
  const bool once = (int64_t)a.S * a.T * a.V * (int64_t)sizeof(T) >= kStreamBytes;
#define RK_BWD(TPR, ONCE)                                                                                             \
  rows_bwd_kernel<T, TPR, ONCE><<<grid_of(a, TPR == rk::kWave), kThreads, 0, st>>>(a, (const T *)x, (const float2 *)stat, g_loss, slope, \
                                                                 g_logps, average, used, (T *)dx)
  if (a.part_len <= kWaveBwd) {
    if (once)
      RK_BWD(rk::kWave, true);
    else
      RK_BWD(rk::kWave, false);
  } else if (once) {
    RK_BWD(kThreads, true);
  } else {
    RK_BWD(kThreads, false);
  }
#undef RK_BWD
  RK_CHECK_LAUNCH("rows_bwd_kernel");
  return RK_OK;
}

}  // namespace

extern "C" {

size_t rk_list_logps_ws_bytes(int32_t S, int32_t T, int32_t V) {
  if (S <= 0 || T <= 0 || V <= 0) return 0;
  Rows a = {0, 0, S, T, V, 0, 0, nullptr, 0, 0, 0};
  cut(a, kWantFwd);
  return (size_t)ws_of(a).words * 4;
}

#define RK_BY_TYPE(fn, ...)                               \
  (dtype == RK_F32 ? fn<float>(__VA_ARGS__)               \
                   : dtype == RK_BF16 ? fn<__bf16>(__VA_ARGS__) : fn<_Float16>(__VA_ARGS__))

int rk_list_logps_fwd(const void *scores, int32_t dtype, int32_t S, int32_t T, int32_t V, int64_t stride_s,
                      int64_t stride_t, const int64_t *items, int64_t ld_items, int64_t ignore_index, int32_t average,
                      float *stat, float *logps, int32_t *used, void *ws, size_t ws_bytes, void *stream) {
  Rows a;
  if (int rc = make_rows(a, dtype, S, T, V, stride_s, stride_t, items, ld_items, ignore_index, kWantFwd)) return rc;
  RK_CHECK_ARG(S == 0 || T > 0, "lists without places");
  if (S == 0) return RK_OK;
  RK_CHECK_ARG(scores && stat && logps && used && ws, "null pointer");
  RK_CHECK_ARG(aligned8(stat) && aligned8(ws), "stat and workspace must be 8-byte aligned");
  RK_CHECK_ARG(ws_bytes >= rk_list_logps_ws_bytes(S, T, V), "workspace too small");
  return RK_BY_TYPE(run_lists, a, scores, average, stat, logps, used, (float *)ws, (hipStream_t)stream);
}

int rk_preference_fwd(const void *scores, int32_t dtype, int32_t S, int32_t T, int32_t V, int64_t stride_s,
                      int64_t stride_t, const int64_t *items, int64_t ld_items, int64_t ignore_index, int32_t average,
                      const float *ref_logps, float beta, float label_smoothing, int32_t kind, float *stat, float *logps,
                      int32_t *used, float *slope, float *loss, void *ws, size_t ws_bytes, void *stream) {
  Rows a;
  if (int rc = make_rows(a, dtype, S, T, V, stride_s, stride_t, items, ld_items, ignore_index, kWantFwd)) return rc;
  RK_CHECK_ARG(S >= 2 && S % 2 == 0 && T > 0, "pairs of lists are needed: %d lists of %d places", S, T);
  RK_CHECK_ARG(kind == RK_PREF_SIGMOID || kind == RK_PREF_HINGE || kind == RK_PREF_SQUARED, "unknown kind %d", kind);
  RK_CHECK_ARG(beta > 0.0f, "beta must be positive");
  RK_CHECK_ARG(label_smoothing >= 0.0f && label_smoothing <= 1.0f, "label smoothing outside [0, 1]");
  RK_CHECK_ARG(label_smoothing == 0.0f || kind == RK_PREF_SIGMOID, "label smoothing is part of the sigmoid form only");
  RK_CHECK_ARG(scores && ref_logps && stat && logps && used && slope && loss && ws, "null pointer");
  RK_CHECK_ARG(aligned8(stat) && aligned8(ws), "stat and workspace must be 8-byte aligned");
  RK_CHECK_ARG(ws_bytes >= rk_list_logps_ws_bytes(S, T, V), "workspace too small");
  return RK_BY_TYPE(run_pairs, a, scores, ref_logps, average, beta, label_smoothing, kind, stat, logps, used, slope, loss,
                    (float *)ws, (hipStream_t)stream);
}

int rk_list_logps_bwd(const void *scores, int32_t dtype, int32_t S, int32_t T, int32_t V, int64_t stride_s,
                      int64_t stride_t, const int64_t *items, int64_t ld_items, int64_t ignore_index, int32_t average,
                      const float *stat, const int32_t *used, const float *g_loss, const float *slope,
                      const float *g_logps, void *d_scores, void *stream) {
  Rows a;
  if (int rc = make_rows(a, dtype, S, T, V, stride_s, stride_t, items, ld_items, ignore_index, kWantBwd)) return rc;
  if (S == 0 || T == 0) return RK_OK;
  RK_CHECK_ARG(scores && stat && used && d_scores, "null pointer");
  RK_CHECK_ARG(aligned8(stat), "stat must be 8-byte aligned");
  RK_CHECK_ARG(!g_loss || slope, "the gradient of the loss needs the slopes of rk_preference_fwd");
  return RK_BY_TYPE(run_bwd, a, scores, stat, g_loss, slope, g_logps, average, used, d_scores, (hipStream_t)stream);
}

}  // extern "C"
