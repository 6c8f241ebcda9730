// Rows of any width: N consecutive elements at any element address (rows of an odd width start off 16-byte boundaries;
// global loads and stores of 4 to 16 bytes take any element address), as floats and back.
#pragma once

#include "common.h"

namespace vk {

typedef float f32x4_e __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x4_e __attribute__((ext_vector_type(4), aligned(2)));
typedef uint16_t u16x8_e __attribute__((ext_vector_type(8), aligned(2)));
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));

// 16 bytes of a row as they are, of data that is read once (past the caches' other contents: a plain read of 179 MB takes
// 29 us, this one 26.5).
__device__ __forceinline__ u32x4 stream_16(const bf16_t *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4_at2 *>(p));
}
__device__ __forceinline__ u32x4 stream_16(const float *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4_at4 *>(p));
}

template <int N>
__device__ __forceinline__ void load_row(const float *p, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const f32x4_e a = *reinterpret_cast<const f32x4_e *>(p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[i + k] = a[k];
  }
}
template <int N>
__device__ __forceinline__ void load_row(const bf16_t *p, float (&v)[N]) {
  if constexpr (N == 8) {
    const u16x8_e a = *reinterpret_cast<const u16x8_e *>(p);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = bf2f(a[k]);
  } else {
    const u16x4_e a = *reinterpret_cast<const u16x4_e *>(p);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = bf2f(a[k]);
  }
}
template <int N>
__device__ __forceinline__ void store_row(float *p, const float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) *reinterpret_cast<f32x4_e *>(p + i) = f32x4_e{v[i], v[i + 1], v[i + 2], v[i + 3]};
}
template <int N>
__device__ __forceinline__ void store_row(bf16_t *p, const float (&v)[N]) {
  typedef uint32_t words_e __attribute__((ext_vector_type(N / 2), aligned(2)));
  words_e o;
#pragma unroll
  for (int k = 0; k < N / 2; ++k) o[k] = pack_bf(v[2 * k], v[2 * k + 1]);
  *reinterpret_cast<words_e *>(p) = o;
}
template <int N>
__device__ __forceinline__ void stream_row(const float *p, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const u32x4 a = stream_16(p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[i + k] = __uint_as_float(a[k]);
  }
}
// store_row of data that is not read again soon.
template <int N>
__device__ __forceinline__ void stream_out(float *p, const float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4)
    __builtin_nontemporal_store(f32x4_e{v[i], v[i + 1], v[i + 2], v[i + 3]}, reinterpret_cast<f32x4_e *>(p + i));
}
template <int N>
__device__ __forceinline__ void stream_out(bf16_t *p, const float (&v)[N]) {
  typedef uint32_t words_e __attribute__((ext_vector_type(N / 2), aligned(2)));
  words_e o;
#pragma unroll
  for (int k = 0; k < N / 2; ++k) o[k] = pack_bf(v[2 * k], v[2 * k + 1]);
  __builtin_nontemporal_store(o, reinterpret_cast<words_e *>(p));
}
__device__ __forceinline__ float load_one(const float *p) { return *p; }
__device__ __forceinline__ float load_one(const bf16_t *p) { return bf2f(*p); }
__device__ __forceinline__ void store_one(float *p, float v) { *p = v; }
__device__ __forceinline__ void store_one(bf16_t *p, float v) { *p = f2bf(v); }

}  // namespace vk
