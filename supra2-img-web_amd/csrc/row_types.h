// float32 values of the row tensors' types (float32, float16, bfloat16), and back with one rounding to nearest even.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sa {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Elements are read and written N at a time through their bytes: one access where N elements are 4, 8 or 16 bytes
// (aligned so), several of 16 bytes beyond. ALIGNED false: one element at a time.

template <int BYTES>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[BYTES / 4]) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const u4 x = reinterpret_cast<const u4*>(p)[i];
      w[4 * i] = x[0], w[4 * i + 1] = x[1], w[4 * i + 2] = x[2], w[4 * i + 3] = x[3];
    }
  } else if constexpr (BYTES == 8) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x, w[1] = x.y;
  } else {
    static_assert(BYTES == 4, "4, 8 or a multiple of 16 bytes");
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

template <int BYTES>
__device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[BYTES / 4]) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) reinterpret_cast<u4*>(p)[i] = u4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
  } else if constexpr (BYTES == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
    static_assert(BYTES == 4, "4, 8 or a multiple of 16 bytes");
    *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
  return (float)x;
}
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  return (T)x;
}

template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ void load_row(const T* p, float (&x)[N]) {
  if constexpr (ALIGNED && (N * sizeof(T)) % 4 == 0) {
    uint32_t w[N * sizeof(T) / 4];
    load_words<N * sizeof(T)>(p, w);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = to_f32(__builtin_bit_cast(T, (uint16_t)(w[i / 2] >> (16 * (i & 1)))));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32(p[i]);
  }
}

template <typename T, int N, bool ALIGNED>
__device__ __forceinline__ void store_row(T* p, const float (&x)[N]) {
  if constexpr (ALIGNED && (N * sizeof(T)) % 4 == 0) {
    uint32_t w[N * sizeof(T) / 4];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = __float_as_uint(x[i]);
    } else {
      typedef T T2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x[2 * i], x[2 * i + 1]}), T2));
    }
    store_words<N * sizeof(T)>(p, w);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from_f32<T>(x[i]);
  }
}

}  // namespace sa
