// V neighbouring elements moved at once, and the sigmoid, for kernels whose vector width follows
// the alignment of their tensors.
#pragma once

#include "dpk_common.h"

#if defined(__HIPCC__)

// V neighbouring elements as loaded, and as floats.
template <typename T, int V> struct vec_io;
template <int V> struct vec_io<float, V> {
  typedef float raw __attribute__((ext_vector_type(V)));
  static __device__ __forceinline__ raw load(const float* p) { return *reinterpret_cast<const raw*>(p); }
  static __device__ __forceinline__ float get(raw r, int j) { return r[j]; }
  static __device__ __forceinline__ void store(float* p, const float* v) {
    raw r;
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = v[j];
    *reinterpret_cast<raw*>(p) = r;
  }
};
template <> struct vec_io<float, 1> {
  typedef float raw;
  static __device__ __forceinline__ raw load(const float* p) { return *p; }
  static __device__ __forceinline__ float get(raw r, int) { return r; }
  static __device__ __forceinline__ void store(float* p, const float* v) { *p = v[0]; }
};
template <int V> struct vec_io<bf16_t, V> {
  typedef uint32_t raw __attribute__((ext_vector_type(V / 2)));
  static __device__ __forceinline__ raw load(const bf16_t* p) { return *reinterpret_cast<const raw*>(p); }
  static __device__ __forceinline__ float get(raw r, int j) {
    const uint32_t w = r[j >> 1];
    return __uint_as_float((j & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ void store(bf16_t* p, const float* v) {
    raw r;
#pragma unroll
    for (int j = 0; j < V / 2; ++j) r[j] = f32x2_to_bf16x2(v[2 * j], v[2 * j + 1]);
    *reinterpret_cast<raw*>(p) = r;
  }
};
template <> struct vec_io<bf16_t, 2> {
  typedef uint32_t raw;
  static __device__ __forceinline__ raw load(const bf16_t* p) { return *reinterpret_cast<const uint32_t*>(p); }
  static __device__ __forceinline__ float get(raw w, int j) {
    return __uint_as_float(j ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ void store(bf16_t* p, const float* v) {
    *reinterpret_cast<uint32_t*>(p) = f32x2_to_bf16x2(v[0], v[1]);
  }
};
template <> struct vec_io<bf16_t, 1> {
  typedef bf16_t raw;
  static __device__ __forceinline__ raw load(const bf16_t* p) { return *p; }
  static __device__ __forceinline__ float get(raw r, int) { return bf16_to_f32(r); }
  static __device__ __forceinline__ void store(bf16_t* p, const float* v) { *p = f32_to_bf16(v[0]); }
};

constexpr float kLog2e = 1.44269504088896340736f;

// 1 / (1 + exp(-v)); 0 and 1 at the infinities. Hardware exp2 and reciprocal, each within 1 ulp.
__device__ __forceinline__ float sigmoid_f(float v) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-v * kLog2e));
}

#endif  // __HIPCC__
