// AdamW over a list of tensors in two launches, with 32-bit or 8-bit moments, parameters and gradients
// in fp32, bfloat16 or fp16, several parameter groups and global-norm clipping (gfx950).
//
//   g = coef * grad                      coef = min(1, max_norm / (|grad| + 1e-6)) over all tensors
//   m = beta1 m + (1 - beta1) g          v = beta2 v + (1 - beta2) g^2
//   p = p - lr wd p - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// Launch 1 advances the step count, adds up the squared gradients (in 64 bits, when clipping is asked
// for; the workgroup that finishes last joins the partial sums in order) and leaves the step's factors
// in the workspace.  Launch 2 updates.  The descriptors travel by value in the kernels' arguments
// (kMaxTensors per launch): nothing is copied or allocated, so a step can be recorded in a HIP graph.
//
// 8-bit moments: blocks of 64 consecutive elements share an fp32 scale; m and the root of v are held as
// e4m3 values, the block's largest magnitude at 448, rounded to nearest.  The root, not v: e4m3 spans
// 2^17.8, which for v would lose every element whose gradients are 480 times smaller than its block's
// largest (a root that is not zero is kept at the smallest code, so that no update divides by eps
// alone).  Blocks of 64, not 256: the block is a row of a 64-wide table, so that a row that is rarely
// touched is not scaled by its busy neighbours.  Update direction against 32-bit moments, cosine over
// simulated steps (spread of the elements' scales e^1; rows touched at rates .5 to .005): 0.986 / 0.994
// with blocks of 64, 0.991 / 0.929 with 256; v itself in e4m3, spread e^2: 0.93.
// All arithmetic is fp32 in a fixed order, without contraction, so the codes are reproducible.
#include <algorithm>

#include "elem.h"

namespace {

constexpr int kMaxTensors = 48;
constexpr int kMaxGroups = RK_ADAMW_MAX_GROUPS;
constexpr int kChunk = 4096;         // elements of a workgroup of the update
constexpr int kNormBlocks = 1024;    // workgroups of the squared-norm launch
constexpr int kBlock = RK_ADAMW_BLOCK;
constexpr float kFull = 448.0f;      // largest finite e4m3 value
constexpr float kTiny = 1e-30f;      // block maxima below this count as this

struct Tensor {
  void *param;
  const void *grad;
  void *m, *v;
  float *m_scale, *v_scale;          // 8-bit moments; NULL: fp32 moments
  int64_t n;
  int32_t kind, group;               // kind: param dtype | grad dtype << 2
};

struct Args {
  Tensor t[kMaxTensors];
  int32_t chunk_start[kMaxTensors + 1];
  int32_t n;
};

struct Hyper {                        // of every group, for the update
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps;
};
struct Hypers {
  Hyper g[kMaxGroups];
};

struct GroupIn {                      // of every group, for the factors
  double beta1, beta2, weight_decay;
};
struct GroupsIn {
  GroupIn g[kMaxGroups];
  int32_t n;
};

struct Factors {                      // what launch 1 leaves for launch 2
  float coef;
  float step_size[kMaxGroups], inv_root_bc2[kMaxGroups], decay[kMaxGroups];
};

__device__ __forceinline__ void write_factors(const GroupsIn &gr, const float *__restrict__ lr, int64_t t, double norm,
                                              float max_norm, float *__restrict__ norm_out, Factors *__restrict__ f) {
  // 1 - beta^t in 64 bits: in 32 it has lost four digits in the first steps
  for (int g = threadIdx.x; g < gr.n; g += (int)blockDim.x) {
    f->step_size[g] = (float)((double)lr[g] / (1.0 - pow(gr.g[g].beta1, (double)t)));
    f->inv_root_bc2[g] = (float)(1.0 / sqrt(1.0 - pow(gr.g[g].beta2, (double)t)));
    f->decay[g] = (float)((double)lr[g] * gr.g[g].weight_decay);
  }
  if (threadIdx.x == 0) {
    const double q = (double)max_norm / (norm + 1e-6);
    f->coef = max_norm > 0.0f && !(q >= 1.0) ? (float)q : 1.0f;   // (a norm that is not a number reaches every element)
    if (norm_out && max_norm > 0.0f) norm_out[0] = (float)norm;
  }
}

__global__ __launch_bounds__(64) void adamw_begin_kernel(GroupsIn gr, const float *__restrict__ lr,
                                                         int64_t *__restrict__ step, Factors *__restrict__ f) {
  const int64_t t = step[0] + 1;
  __syncthreads();
  if (threadIdx.x == 0) step[0] = t;
  write_factors(gr, lr, t, 0.0, 0.0f, nullptr, f);
}

template <typename T>
__device__ __forceinline__ double square_sum(const T *__restrict__ g, int64_t lo, int64_t hi) {
  constexpr int VEC = rk::Elem<T>::kVec;
  double s = 0.0;
  int64_t i = lo + (int64_t)threadIdx.x * VEC;
  for (; i + VEC <= hi; i += 256 * VEC) {
    rk::Pack<T, VEC> v;
    v.load(g + i);
    float f[VEC];
    v.widen(f);
#pragma unroll
    for (int e = 0; e < VEC; ++e) s = fma((double)f[e], (double)f[e], s);
  }
  for (int e = 0; e < VEC && i + e < hi; ++e) {
    const double x = (double)rk::Elem<T>::get(g[i + e]);
    s = fma(x, x, s);
  }
  return s;
}

__device__ __forceinline__ int find_tensor(const Args &a, int32_t chunk) {
  int i = 0;
  while (i + 1 < a.n && a.chunk_start[i + 1] <= chunk) ++i;
  return i;
}

// Squared gradients of one launch's tensors, one partial sum per workgroup; the last workgroup of the
// last launch (n_partial > 0) joins all of them in order and writes the factors.  The partial sums are
// stored and read with agent scope around the ticket: the workgroups run under different L2 caches.
__global__ __launch_bounds__(256) void adamw_norm_kernel(Args a, double *__restrict__ partial, int32_t first,
                                                         int32_t n_partial, int32_t *__restrict__ ticket, GroupsIn gr,
                                                         const float *__restrict__ lr, int64_t *__restrict__ step,
                                                         float max_norm, float *__restrict__ norm_out,
                                                         Factors *__restrict__ f) {
  __shared__ double red[4];
  __shared__ int s_last;
  double s = 0.0;
  const int32_t chunks = a.chunk_start[a.n];
  for (int32_t c = blockIdx.x; c < chunks; c += (int32_t)gridDim.x) {
    const int i = find_tensor(a, c);
    const Tensor &t = a.t[i];
    const int64_t lo = (int64_t)(c - a.chunk_start[i]) * kChunk, hi = min(t.n, lo + kChunk);
    const int gd = t.kind >> 2;
    if (gd == RK_F32)
      s += square_sum((const float *)t.grad, lo, hi);
    else if (gd == RK_BF16)
      s += square_sum((const __bf16 *)t.grad, lo, hi);
    else
      s += square_sum((const _Float16 *)t.grad, lo, hi);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, rk::kWave);
  if (threadIdx.x % rk::kWave == 0) red[threadIdx.x / rk::kWave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    __hip_atomic_store(&partial[first + blockIdx.x], (red[0] + red[1]) + (red[2] + red[3]), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
    __threadfence();
    s_last = n_partial > 0 &&
             __hip_atomic_fetch_add(ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int32_t)gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double all = 0.0;
  for (int32_t i = threadIdx.x; i < n_partial; i += 256)
    all += __hip_atomic_load(&partial[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) all += __shfl_xor(all, off, rk::kWave);
  if (threadIdx.x % rk::kWave == 0) red[threadIdx.x / rk::kWave] = all;
  const int64_t t = step[0] + 1;
  __syncthreads();
  if (threadIdx.x == 0) {
    step[0] = t;
    ticket[0] = 0;                    // ready for the next step
  }
  write_factors(gr, lr, t, sqrt((red[0] + red[1]) + (red[2] + red[3])), max_norm, norm_out, f);
}

// largest value of a row of 16 lanes, in all of them
__device__ __forceinline__ float row_max16(float x) {
#define RK_ROW_MAX(CTRL) \
  x = fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), CTRL, 0xF, 0xF, false)))
  RK_ROW_MAX(0x128);   // row_ror:8
  RK_ROW_MAX(0x124);
  RK_ROW_MAX(0x122);
  RK_ROW_MAX(0x121);
#undef RK_ROW_MAX
  return x;
}

__device__ __forceinline__ uint32_t encode4(const float (&x)[4]) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
}
__device__ __forceinline__ void decode4(uint32_t w, float scale, float (&x)[4]) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo[0] * scale;
  x[1] = lo[1] * scale;
  x[2] = hi[0] * scale;
  x[3] = hi[1] * scale;
}

// Four consecutive elements per lane and step: 16 lanes hold one block of 64.
template <typename PT, typename GT, bool Q8>
__device__ __forceinline__ void update(const Tensor &t, int64_t lo, int64_t hi, const Hyper &h, const Factors &f, int group) {
  constexpr int U = kChunk / 1024;
  PT *__restrict__ P = (PT *)t.param;
  const GT *__restrict__ G = (const GT *)t.grad;
  float p[U][4], g[U][4], m[U][4], v[U][4];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = lo + u * 1024 + (int64_t)threadIdx.x * 4;
    if (i + 4 <= hi) {
      rk::Pack<PT, 4> a;
      a.load(P + i);
      a.widen(p[u]);
      rk::Pack<GT, 4> b;
      b.load(G + i);
      b.widen(g[u]);
      if constexpr (!Q8) {
        rk::Pack<float, 4> c;
        c.load((const float *)t.m + i);
        c.widen(m[u]);
        c.load((const float *)t.v + i);
        c.widen(v[u]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = i + e < hi;
        p[u][e] = in ? rk::Elem<PT>::get(P[i + e]) : 0.0f;
        g[u][e] = in ? rk::Elem<GT>::get(G[i + e]) : 0.0f;
        if constexpr (!Q8) {
          m[u][e] = in ? ((const float *)t.m)[i + e] : 0.0f;
          v[u][e] = in ? ((const float *)t.v)[i + e] : 0.0f;
        }
      }
    }
    if constexpr (Q8) {
      if (i < hi) {                   // (the codes are padded to whole blocks)
        const int64_t b = i / kBlock;
        decode4(((const uint32_t *)t.m)[i / 4], t.m_scale[b], m[u]);
        decode4(((const uint32_t *)t.v)[i / 4], t.v_scale[b], v[u]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[u][e] *= v[u][e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) m[u][e] = v[u][e] = 0.0f;
      }
    }
  }
  const float coef = f.coef, step_size = f.step_size[group], inv_root = f.inv_root_bc2[group], decay = f.decay[group];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = lo + u * 1024 + (int64_t)threadIdx.x * 4;
    float r[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = g[u][e] * coef;
      m[u][e] = m[u][e] * h.beta1 + x * h.one_minus_beta1;
      v[u][e] = v[u][e] * h.beta2 + (x * x) * h.one_minus_beta2;
      r[e] = sqrtf(v[u][e]);
      // (the reciprocal is good to one unit in the last place, and the update is small beside p)
      const float q = p[u][e] - p[u][e] * decay;
      p[u][e] = q - step_size * (m[u][e] * __builtin_amdgcn_rcpf(r[e] * inv_root + h.eps));
    }
    if (i + 4 <= hi) {
      rk::Pack<PT, 4> a;
      a.narrow(p[u]);
      a.store(P + i);
      if constexpr (!Q8) {
        rk::Pack<float, 4> c;
        c.narrow(m[u]);
        c.store((float *)t.m + i);
        c.narrow(v[u]);
        c.store((float *)t.v + i);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (i + e >= hi) {
          m[u][e] = r[e] = 0.0f;
          continue;
        }
        P[i + e] = rk::Elem<PT>::put(p[u][e]);
        if constexpr (!Q8) {
          ((float *)t.m)[i + e] = m[u][e];
          ((float *)t.v)[i + e] = v[u][e];
        }
      }
    }
    if constexpr (Q8) {
      // (every lane of a row takes part in its maximum, those behind the end with zeros)
      const float am = fmaxf(row_max16(fmaxf(fmaxf(fabsf(m[u][0]), fabsf(m[u][1])), fmaxf(fabsf(m[u][2]), fabsf(m[u][3])))), kTiny);
      const float ar = fmaxf(row_max16(fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]))), kTiny);
      const float im = (1.0f / am) * kFull, ir = (1.0f / ar) * kFull;
      float x[4], y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = m[u][e] * im;
        y[e] = r[e] * ir;
        if (r[e] > 0.0f) y[e] = fmaxf(y[e], 0.001953125f);   // 2^-9, the smallest code above zero
      }
      if (i < hi) {
        ((uint32_t *)t.m)[i / 4] = encode4(x);
        ((uint32_t *)t.v)[i / 4] = encode4(y);
        if (threadIdx.x % 16 == 0) {
          t.m_scale[i / kBlock] = am * (1.0f / kFull);
          t.v_scale[i / kBlock] = ar * (1.0f / kFull);
        }
      }
    }
  }
}

__global__ __launch_bounds__(256) void adamw_update_kernel(Args a, Hypers hy, const Factors *__restrict__ fp) {
  const int k = find_tensor(a, (int32_t)blockIdx.x);
  const Tensor &t = a.t[k];
  const int64_t lo = (int64_t)((int32_t)blockIdx.x - a.chunk_start[k]) * kChunk, hi = min(t.n, lo + kChunk);
  const Factors &f = *fp;
  const Hyper &h = hy.g[t.group];
#define RK_CASE(PD, GD, PT, GT)                           \
  case (PD) | (GD) << 2:                                  \
    if (t.m_scale)                                        \
      update<PT, GT, true>(t, lo, hi, h, f, t.group);     \
    else                                                  \
      update<PT, GT, false>(t, lo, hi, h, f, t.group);    \
    break;
  switch (t.kind) {
    RK_CASE(RK_F32, RK_F32, float, float)
    RK_CASE(RK_BF16, RK_BF16, __bf16, __bf16)
    RK_CASE(RK_BF16, RK_F32, __bf16, float)
    RK_CASE(RK_F16, RK_F16, _Float16, _Float16)
    RK_CASE(RK_F16, RK_F32, _Float16, float)
  }
#undef RK_CASE
}

int launches_of(int32_t n_tensors) { return (int)rk::ceil_div(n_tensors, kMaxTensors); }

// workspace: factors, ticket, partial sums
constexpr size_t kTicketAt = (sizeof(Factors) + 15) / 16 * 16, kPartialAt = kTicketAt + 16;

}  // namespace

extern "C" {

size_t rk_adamw_ws_bytes(int32_t n_tensors) {
  if (n_tensors <= 0) return 0;
  return kPartialAt + (size_t)launches_of(n_tensors) * kNormBlocks * sizeof(double);
}

int rk_adamw_step(const rk_adamw_tensor *tensors_host, int32_t n_tensors, const rk_adamw_group *groups_host,
                  int32_t n_groups, int64_t *step, const float *lr, float max_norm, float *norm_out, void *ws,
                  size_t ws_bytes, void *stream) {
  RK_CHECK_ARG(n_tensors >= 0, "negative tensor count");
  if (n_tensors == 0) return RK_OK;
  RK_CHECK_ARG(tensors_host && groups_host && step && lr && ws, "null pointer");
  RK_CHECK_ARG(n_groups >= 1 && n_groups <= kMaxGroups, "%d parameter groups: 1 to %d are built", n_groups, kMaxGroups);
  RK_CHECK_ARG(ws_bytes >= rk_adamw_ws_bytes(n_tensors) && rk::aligned16(ws), "workspace too small or not aligned");
  GroupsIn gr = {};
  Hypers hy = {};
  gr.n = n_groups;
  for (int g = 0; g < n_groups; ++g) {
    const rk_adamw_group &s = groups_host[g];
    RK_CHECK_ARG(s.beta1 >= 0.0 && s.beta1 < 1.0 && s.beta2 >= 0.0 && s.beta2 < 1.0 && s.eps >= 0.0 && s.weight_decay >= 0.0,
                 "group %d: bad AdamW constants", g);
    gr.g[g] = {s.beta1, s.beta2, s.weight_decay};
    hy.g[g] = {(float)s.beta1, (float)(1.0 - s.beta1), (float)s.beta2, (float)(1.0 - s.beta2), (float)s.eps};
  }
  int64_t chunks = 0;
  for (int i = 0; i < n_tensors; ++i) {
    const rk_adamw_tensor &t = tensors_host[i];
    RK_CHECK_ARG(t.n > 0 && t.param && t.grad && t.exp_avg && t.exp_avg_sq, "tensor %d: null pointer or empty", i);
    RK_CHECK_ARG(!t.exp_avg_scale == !t.exp_avg_sq_scale, "tensor %d: one of the two scales is missing", i);
    RK_CHECK_ARG(t.group >= 0 && t.group < n_groups, "tensor %d: group %d outside [0, %d)", i, t.group, n_groups);
    const int pd = t.param_dtype, gd = t.grad_dtype;
    RK_CHECK_ARG(pd == RK_F32 || pd == RK_BF16 || pd == RK_F16, "tensor %d: unknown element type %d", i, pd);
    RK_CHECK_ARG(gd == pd || gd == RK_F32, "tensor %d: gradients have the parameter's type or fp32", i);
    // (codes are read four at a time)
    RK_CHECK_ARG(!t.exp_avg_scale || (((uintptr_t)t.exp_avg | (uintptr_t)t.exp_avg_sq) & 3) == 0,
                 "tensor %d: 8-bit moments must be 4-byte aligned", i);
    chunks += rk::ceil_div(t.n, kChunk);
  }
  RK_CHECK_ARG(chunks < INT32_MAX, "too many elements");
  hipStream_t st = (hipStream_t)stream;
  Factors *f = (Factors *)ws;
  int32_t *ticket = (int32_t *)((char *)ws + kTicketAt);
  double *partial = (double *)((char *)ws + kPartialAt);
  const bool clip = max_norm > 0.0f;
  if (!clip) {
    adamw_begin_kernel<<<1, 64, 0, st>>>(gr, lr, step, f);
    RK_CHECK_LAUNCH("adamw_begin_kernel");
  }
  const int launches = launches_of(n_tensors);
  for (int pass = clip ? 0 : 1; pass < 2; ++pass) {
    int32_t first = 0;
    for (int l = 0; l < launches; ++l) {
      Args a;
      a.n = std::min(kMaxTensors, n_tensors - l * kMaxTensors);
      int32_t c = 0;
      for (int i = 0; i < a.n; ++i) {
        const rk_adamw_tensor &t = tensors_host[l * kMaxTensors + i];
        a.t[i] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale, t.exp_avg_sq_scale, t.n,
                  t.param_dtype | t.grad_dtype << 2, t.group};
        a.chunk_start[i] = c;
        c += (int32_t)rk::ceil_div(t.n, kChunk);
      }
      a.chunk_start[a.n] = c;
      if (pass == 0) {
        const int32_t blocks = std::min(c, kNormBlocks);
        const int32_t joined = l + 1 == launches ? first + blocks : 0;
        adamw_norm_kernel<<<blocks, 256, 0, st>>>(a, partial, first, joined, ticket, gr, lr, step, max_norm, norm_out, f);
        RK_CHECK_LAUNCH("adamw_norm_kernel");
        first += blocks;
      } else {
        adamw_update_kernel<<<c, 256, 0, st>>>(a, hy, f);
        RK_CHECK_LAUNCH("adamw_update_kernel");
      }
    }
  }
  return RK_OK;
}

}  // extern "C"
