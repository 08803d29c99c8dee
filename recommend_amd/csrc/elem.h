// Element types of the kernels that take fp32, bfloat16 and fp16 tensors (RK_F32, RK_BF16, RK_F16):
// 16-byte vectors in memory, fp32 in registers, one rounding (to nearest even) on the way out.
#pragma once
#include "common.h"

namespace rk {

typedef uint32_t u32x4_at_elem __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));

template <typename T>
struct Elem;

template <>
struct Elem<float> {
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
  static __device__ __forceinline__ void widen(uint32_t w, float *o) { o[0] = __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t narrow(const float *x) { return __float_as_uint(x[0]); }
};

template <>
struct Elem<__bf16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(__bf16 x) { return (float)x; }
  static __device__ __forceinline__ __bf16 put(float x) { return (__bf16)x; }
  static __device__ __forceinline__ void widen(uint32_t w, float *o) {
    o[0] = __uint_as_float(w << 16);
    o[1] = __uint_as_float(w & 0xFFFF0000u);
  }
  static __device__ __forceinline__ uint32_t narrow(const float *x) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v{x[0], x[1]}), bf16x2v));
  }
};

template <>
struct Elem<_Float16> {
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(_Float16 x) { return (float)x; }
  static __device__ __forceinline__ _Float16 put(float x) { return (_Float16)x; }
  static __device__ __forceinline__ void widen(uint32_t w, float *o) {
    const f32x2v v = __builtin_convertvector(__builtin_bit_cast(f16x2v, w), f32x2v);
    o[0] = v[0];
    o[1] = v[1];
  }
  static __device__ __forceinline__ uint32_t narrow(const float *x) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v{x[0], x[1]}), f16x2v));
  }
};

// N elements from an address that is aligned to ONE element only: gfx950 reads and writes unaligned
// vectors in global memory, so a row of odd length needs no scalar prologue.
template <typename T, int N>
struct Pack {
  static constexpr int kBytes = N * (int)sizeof(T);
  static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T *p) { __builtin_memcpy(w, p, kBytes); }
  __device__ __forceinline__ void store(T *p) const { __builtin_memcpy(p, w, kBytes); }
  // the same for data that is touched once: it does not push other data out of the caches
  __device__ __forceinline__ void load_once(const T *p) {
    if constexpr (kWords == 4) {
      const u32x4_at_elem v = __builtin_nontemporal_load((const u32x4_at_elem *)p);
      __builtin_memcpy(w, &v, 16);
    } else {
      load(p);
    }
  }
  __device__ __forceinline__ void store_once(T *p) const {
    if constexpr (kWords == 4) {
      u32x4_at_elem v;
      __builtin_memcpy(&v, w, 16);
      __builtin_nontemporal_store(v, (u32x4_at_elem *)p);
    } else {
      store(p);
    }
  }
  __device__ __forceinline__ void widen(float (&o)[N]) const {
    if constexpr (kBytes < 4) {
      T x;
      __builtin_memcpy(&x, w, kBytes);
      o[0] = Elem<T>::get(x);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) Elem<T>::widen(w[i], o + i * (4 / (int)sizeof(T)));
    }
  }
  __device__ __forceinline__ void narrow(const float (&x)[N]) {
    if constexpr (kBytes < 4) {
      const T v = Elem<T>::put(x[0]);
      __builtin_memcpy(w, &v, kBytes);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = Elem<T>::narrow(x + i * (4 / (int)sizeof(T)));
    }
  }
};

// workgroups of 256 threads in one dimension of a grid, which is counted in threads, in 32 bits
constexpr int64_t kMaxBlocks256 = (1ll << 32) / 256 - 1;

}  // namespace rk
