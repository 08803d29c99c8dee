// AdamW over a list of tensors in two or three launches, with 32-bit or 8-bit moments, parameters and gradients
// in fp32, bfloat16 or fp16, several parameter groups and global-norm clipping (gfx950).
//
//   g = coef * grad                      coef = min(1, max_norm / (|grad| + 1e-6)) over all tensors
//   m = beta1 m + (1 - beta1) g          v = beta2 v + (1 - beta2) g^2
//   p = p - lr wd p - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
//
// Where clipping is asked for, the first launch adds up the squared gradients, in 64 bits, one partial
// sum per workgroup.  The next one, a single workgroup, advances the step count, joins the partial sums
// in order and leaves the step's factors in the workspace.  The last one updates.  (Joining in the
// workgroup that finishes the norm last saves the small launch, but its release fences write back the
// L2 once per workgroup: 158 us instead of 60 for 167 MB.)  The descriptors travel by value in the kernels' arguments
// (kMaxTensors per launch): nothing is copied or allocated, so a step can be recorded in a HIP graph.
//
// 8-bit moments: blocks of 64 consecutive elements share an fp32 scale; m and the root of v are held as
// e4m3 values, the block's largest magnitude at 448, rounded to nearest.  The root, not v: e4m3 spans
// 2^17.8, which for v would lose every element whose gradients are 480 times smaller than its block's
// largest (a root that is not zero is kept at the smallest code, so that no update divides by eps
// alone).  Blocks of 64, not 256: the block is a row of a 64-wide table, so that a row that is rarely
// touched is not scaled by its busy neighbours.  Update direction against 32-bit moments, cosine over
// simulated steps (spread of the elements' scales e^1; rows touched at rates .5 to .005): 0.986 / 0.994
// with blocks of 64, 0.991 / 0.929 with 256; v itself in e4m3, spread e^2: 0.93.  These are steady gradients.
// Rounded to nearest, a root keeps its code until one step moves it by half a code against its block's largest, so
// with beta2 = 0.999 it does not follow a gradient that shrinks against its neighbours': every second element's a tenth
// from step 500 on gives 0.88 at step 2000 and 0.80 at 4000 (beta2 = 0.95: 0.996); a change of a whole block is followed.
// All arithmetic is fp32 in a fixed order, without contraction, so the codes are reproducible.
#include <algorithm>

#include "elem.h"

namespace {

constexpr int kMaxTensors = 48;
constexpr int kMaxGroups = RK_ADAMW_MAX_GROUPS;
constexpr int kChunk = 2048;         // elements of a workgroup of the update
constexpr int kNormVectors = 8;      // 16-byte vectors of a lane that the squared-norm launch has in flight
constexpr int kNormBlocks = 2048;    // its workgroups
constexpr int kBlock = RK_ADAMW_BLOCK;
constexpr float kFull = 448.0f;      // largest finite e4m3 value
constexpr float kTiny = 1e-30f;      // block maxima below this count as this

// elements that a workgroup of the squared-norm launch takes at a time
__host__ __device__ __forceinline__ int norm_chunk(int grad_dtype) {
  return kNormVectors * 256 * (grad_dtype == RK_F32 ? 4 : 8);
}

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

// x^t by squaring: a dozen instructions where pow() costs the kernel a third of its registers
__device__ __forceinline__ double power(double x, int64_t t) {
  double y = 1.0;
  for (; t > 0; t >>= 1, x *= x)
    if (t & 1) y *= x;
  return y;
}

__device__ __forceinline__ void write_factors(const GroupsIn &gr, const float *__restrict__ lr, int64_t t, double norm,
                                              float max_norm, float *__restrict__ norm_out, Factors *__restrict__ f) {
  // 1 - beta^t in 64 bits: in 32 it has lost four digits in the first steps
  for (int g = threadIdx.x; g < gr.n; g += (int)blockDim.x) {
    f->step_size[g] = (float)((double)lr[g] / (1.0 - power(gr.g[g].beta1, t)));
    f->inv_root_bc2[g] = (float)(1.0 / sqrt(1.0 - power(gr.g[g].beta2, t)));
    f->decay[g] = (float)((double)lr[g] * gr.g[g].weight_decay);
  }
  if (threadIdx.x == 0) {
    const double q = (double)max_norm / (norm + 1e-6);
    f->coef = max_norm > 0.0f && !(q >= 1.0) ? (float)q : 1.0f;   // (a norm that is not a number reaches every element)
    if (norm_out && max_norm > 0.0f) norm_out[0] = (float)norm;
  }
}

// One workgroup: the step count, the gradients' norm from the partial sums of the norm launches (in
// order), the step's factors.
__global__ __launch_bounds__(256) void adamw_begin_kernel(GroupsIn gr, const float *__restrict__ lr,
                                                          int64_t *__restrict__ step, const double *__restrict__ partial,
                                                          int32_t n_partial, float max_norm, float *__restrict__ norm_out,
                                                          Factors *__restrict__ f) {
  __shared__ double red[4];
  const int64_t t = step[0] + 1;
  double s = 0.0;
#pragma unroll 8
  for (int32_t i = threadIdx.x; i < n_partial; i += 256) s += partial[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, rk::kWave);
  if (threadIdx.x % rk::kWave == 0) red[threadIdx.x / rk::kWave] = s;
  __syncthreads();
  if (threadIdx.x == 0) step[0] = t;
  write_factors(gr, lr, t, sqrt((red[0] + red[1]) + (red[2] + red[3])), max_norm, norm_out, f);
}

// sum of squares of g[lo .. hi) (a chunk), in 64 bits, all vectors of a lane in flight
template <typename T>
__device__ __forceinline__ double square_sum(const T *__restrict__ g, int64_t lo, int64_t hi) {
  constexpr int VEC = rk::Elem<T>::kVec, U = kNormVectors;
  double s[2] = {0.0, 0.0};
  int64_t i = lo + (int64_t)threadIdx.x * VEC;
  for (; i + (U - 1) * 256 * VEC + VEC <= hi; i += U * 256 * VEC) {
    rk::Pack<T, VEC> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u].load(g + i + u * 256 * VEC);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float f[VEC];
      v[u].widen(f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[e & 1] = fma((double)f[e], (double)f[e], s[e & 1]);
    }
  }
  for (; i < hi; i += 256 * VEC) {
    float f[VEC];
    if (i + VEC <= hi) {
      rk::Pack<T, VEC> v;
      v.load(g + i);
      v.widen(f);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = i + e < hi ? rk::Elem<T>::get(g[i + e]) : 0.0f;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[e & 1] = fma((double)f[e], (double)f[e], s[e & 1]);
  }
  return s[0] + s[1];
}

// Squared gradients of one launch's tensors, one partial sum per workgroup.  Neighbouring workgroups read
// neighbouring chunks: with a consecutive share for each they met on the same memory channels (433 MB in
// 208 us instead of 110).
__global__ __launch_bounds__(256) void adamw_norm_kernel(Args a, double *__restrict__ partial) {
  __shared__ double red[4];
  double s = 0.0;
  const int32_t chunks = a.chunk_start[a.n];
  for (int32_t c = blockIdx.x, i = 0; c < chunks; c += (int32_t)gridDim.x) {
    while (a.chunk_start[i + 1] <= c) ++i;
    const Tensor &t = a.t[i];
    const int gd = t.kind >> 2;
    const int64_t lo = (int64_t)(c - a.chunk_start[i]) * norm_chunk(gd), hi = min(t.n, lo + norm_chunk(gd));
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
  if (threadIdx.x == 0) partial[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// Largest of non-negative floats over a row of 16 lanes, in all of them.  As integers: the order of
// non-negative floats is that of their bits, and a NaN is larger than all (so it reaches the block's
// scale), without the extra instructions that quiet a float maximum's operands.
__device__ __forceinline__ uint32_t row_max16(uint32_t x) {
#define RK_ROW_MAX(CTRL) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xF, 0xF, false))
  RK_ROW_MAX(0x128);   // row_ror:8
  RK_ROW_MAX(0x124);
  RK_ROW_MAX(0x122);
  RK_ROW_MAX(0x121);
#undef RK_ROW_MAX
  return x;
}

// 1 / x and sqrt(x) rounded to nearest in a few instructions: the hardware's approximation and one
// correction with the exact residual.  Equal to the correctly rounded results for every significand
// (checked over all of them, at exponents from -100 to 100); unlike the compiler's expansions they do not
// care for subnormal x, whose roots (below 2^-63) are zero to an update.
__device__ __forceinline__ float exact_rcp(float x) {
  const float y = __builtin_amdgcn_rcpf(x);
  return fmaf(fmaf(-x, y, 1.0f), y, y);
}
__device__ __forceinline__ float exact_sqrt(float x) {
  const float y = __builtin_amdgcn_rsqf(fmaxf(x, 0x1p-126f)), s = x * y;
  return fmaf(fmaf(-s, s, x), 0.5f * y, s);
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

// Four consecutive elements per lane and step: 16 lanes hold one block of 64.  FULL: the whole chunk
// lies in the tensor (i.e. all but a tensor's last).
template <typename PT, typename GT, bool Q8, bool FULL>
__device__ __forceinline__ void update(const Tensor &t, int64_t chunk, const Hyper &h, const Factors &f, int group) {
  constexpr int U = kChunk / 1024;
  const int left = FULL ? kChunk : (int)(t.n - chunk);     // elements of the tensor from the chunk on
  PT *__restrict__ P = (PT *)t.param + chunk;
  const GT *__restrict__ G = (const GT *)t.grad + chunk;
  float *__restrict__ M = (float *)t.m + chunk, *__restrict__ V = (float *)t.v + chunk;
  uint32_t *__restrict__ CM = (uint32_t *)t.m + chunk / 4, *__restrict__ CV = (uint32_t *)t.v + chunk / 4;
  float *__restrict__ SM = t.m_scale + chunk / kBlock, *__restrict__ SV = t.v_scale + chunk / kBlock;
  rk::Pack<PT, 4> p[U];
  rk::Pack<GT, 4> g[U];
  rk::Pack<float, 4> m[U], v[U];
  uint32_t cm[U], cv[U];
  float sm[U], sv[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = u * 1024 + (int)threadIdx.x * 4;
    if (FULL || i + 4 <= left) {
      p[u].load_once(P + i);
      g[u].load_once(G + i);
      if constexpr (!Q8) {
        m[u].load_once(M + i);
        v[u].load_once(V + i);
      }
    } else {
      float x[4], y[4], z[4], w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = i + e < left;
        x[e] = in ? rk::Elem<PT>::get(P[i + e]) : 0.0f;
        y[e] = in ? rk::Elem<GT>::get(G[i + e]) : 0.0f;
        z[e] = !Q8 && in ? M[i + e] : 0.0f;
        w[e] = !Q8 && in ? V[i + e] : 0.0f;
      }
      p[u].narrow(x);
      g[u].narrow(y);
      m[u].narrow(z);
      v[u].narrow(w);
    }
    if constexpr (Q8) {
      const bool in = FULL || i < left;                    // (the codes are padded to whole blocks)
      cm[u] = in ? CM[i / 4] : 0u;
      cv[u] = in ? CV[i / 4] : 0u;
      sm[u] = in ? SM[i / kBlock] : 0.0f;
      sv[u] = in ? SV[i / kBlock] : 0.0f;
    }
  }
  const float coef = f.coef, step_size = f.step_size[group], inv_root = f.inv_root_bc2[group], decay = f.decay[group];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = u * 1024 + (int)threadIdx.x * 4;
    float x[4], d[4], a[4], b[4], r[4];
    p[u].widen(x);
    g[u].widen(d);
    if constexpr (Q8) {
      decode4(cm[u], sm[u], a);
      decode4(cv[u], sv[u], b);
#pragma unroll
      for (int e = 0; e < 4; ++e) b[e] *= b[e];
    } else {
      m[u].widen(a);
      v[u].widen(b);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float y = d[e] * coef;
      a[e] = a[e] * h.beta1 + y * h.one_minus_beta1;
      b[e] = b[e] * h.beta2 + (y * y) * h.one_minus_beta2;
      r[e] = Q8 ? exact_sqrt(b[e]) : sqrtf(b[e]);
      // (fused where the result is only p: rounded once less, and the reciprocal is good to a unit in the last place)
      const float q = fmaf(-x[e], decay, x[e]);
      x[e] = fmaf(-step_size, a[e] * __builtin_amdgcn_rcpf(fmaf(r[e], inv_root, h.eps)), q);
    }
    if (FULL || i + 4 <= left) {
      p[u].narrow(x);
      p[u].store_once(P + i);
      if constexpr (!Q8) {
        m[u].narrow(a);
        m[u].store_once(M + i);
        v[u].narrow(b);
        v[u].store_once(V + i);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (i + e >= left) {
          a[e] = r[e] = 0.0f;
          continue;
        }
        P[i + e] = rk::Elem<PT>::put(x[e]);
        if constexpr (!Q8) {
          M[i + e] = a[e];
          V[i + e] = b[e];
        }
      }
    }
    if constexpr (Q8) {
      // (every lane of a row takes part in its maximum, those behind the end with zeros)
      uint32_t ua[4], ur[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ua[e] = __float_as_uint(a[e]) & 0x7FFFFFFFu;
        ur[e] = __float_as_uint(r[e]) & 0x7FFFFFFFu;
      }
      const uint32_t tiny = __float_as_uint(kTiny);
      const float am = __uint_as_float(max(row_max16(max(max(ua[0], ua[1]), max(ua[2], ua[3]))), tiny));
      const float ar = __uint_as_float(max(row_max16(max(max(ur[0], ur[1]), max(ur[2], ur[3]))), tiny));
      const float im = exact_rcp(am) * kFull, ir = exact_rcp(ar) * kFull;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] *= im;
        // a root above zero gets the smallest code, 2^-9, at least: the median of a huge number, the value and 2^-9
        r[e] = __builtin_amdgcn_fmed3f(r[e] * 0x1p126f, r[e] * ir, 0x1p-9f);
      }
      if (FULL || i < left) {
        CM[i / 4] = encode4(a);
        CV[i / 4] = encode4(r);
        if (threadIdx.x % 16 == 0) {
          SM[i / kBlock] = am * (1.0f / kFull);
          SV[i / kBlock] = ar * (1.0f / kFull);
        }
      }
    }
  }
}

__device__ __forceinline__ int find_tensor(const Args &a, int32_t chunk) {
  int i = 0;
  while (i + 1 < a.n && a.chunk_start[i + 1] <= chunk) ++i;
  return i;
}

__global__ __launch_bounds__(256) void adamw_update_kernel(Args a, Hypers hy, const Factors *__restrict__ fp) {
  const int k = find_tensor(a, (int32_t)blockIdx.x);
  const Tensor &t = a.t[k];
  const int64_t chunk = (int64_t)((int32_t)blockIdx.x - a.chunk_start[k]) * kChunk;
  const Factors &f = *fp;
  const Hyper &h = hy.g[t.group];
  const bool full = chunk + kChunk <= t.n;
#define RK_CASE(PD, GD, PT, GT)                                   \
  case (PD) | (GD) << 2:                                          \
    if (t.m_scale) {                                              \
      if (full)                                                   \
        update<PT, GT, true, true>(t, chunk, h, f, t.group);      \
      else                                                        \
        update<PT, GT, true, false>(t, chunk, h, f, t.group);     \
    } else if (full) {                                            \
      update<PT, GT, false, true>(t, chunk, h, f, t.group);       \
    } else {                                                      \
      update<PT, GT, false, false>(t, chunk, h, f, t.group);      \
    }                                                             \
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

// workspace: factors, partial sums
constexpr size_t kPartialAt = (sizeof(Factors) + 15) / 16 * 16;

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
  int64_t chunks = 0;                 // of the update's current launch
  for (int i = 0; i < n_tensors; ++i) {
    if (i % kMaxTensors == 0) chunks = 0;
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
    RK_CHECK_ARG(chunks < rk::kMaxBlocks256, "too many elements in one launch's tensors");
  }
  hipStream_t st = (hipStream_t)stream;
  Factors *f = (Factors *)ws;
  double *partial = (double *)((char *)ws + kPartialAt);
  const bool clip = max_norm > 0.0f;
  const int launches = launches_of(n_tensors);
  int32_t n_partial = 0;
  for (int pass = clip ? 0 : 1; pass < 2; ++pass) {
    if (pass == 1) {
      adamw_begin_kernel<<<1, 256, 0, st>>>(gr, lr, step, partial, n_partial, max_norm, norm_out, f);
      RK_CHECK_LAUNCH("adamw_begin_kernel");
    }
    for (int l = 0; l < launches; ++l) {
      Args a;
      a.n = std::min(kMaxTensors, n_tensors - l * kMaxTensors);
      int32_t c = 0;
      for (int i = 0; i < a.n; ++i) {
        const rk_adamw_tensor &t = tensors_host[l * kMaxTensors + i];
        a.t[i] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.exp_avg_scale, t.exp_avg_sq_scale, t.n,
                  t.param_dtype | t.grad_dtype << 2, t.group};
        a.chunk_start[i] = c;
        c += (int32_t)rk::ceil_div(t.n, pass == 0 ? norm_chunk(t.grad_dtype) : kChunk);
      }
      a.chunk_start[a.n] = c;
      if (pass == 0) {
        const int32_t blocks = std::min(c, kNormBlocks);
        adamw_norm_kernel<<<blocks, 256, 0, st>>>(a, partial + n_partial);
        RK_CHECK_LAUNCH("adamw_norm_kernel");
        n_partial += blocks;
      } else {
        adamw_update_kernel<<<c, 256, 0, st>>>(a, hy, f);
        RK_CHECK_LAUNCH("adamw_update_kernel");
      }
    }
  }
  return RK_OK;
}

}  // extern "C"
