// A row of V logits (any V, any element address) held or walked by a group of GL consecutive threads: the 16-byte vectors
// between its first and its last 16-byte boundary, vector c GL + lane with thread `lane`, and up to 14 edge elements in
// front of and behind them, one with each of the first threads. What the operators on rows of logits share
// (objectives.hip, top_logits.hip).
#pragma once

#include <math.h>

#include <type_traits>

#include "row_access.h"

namespace vk {

template <typename T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));  // elements of a vector

__device__ __forceinline__ float vec_at(const u32x4 &r, int k, const bf16_t *) {
  return (k & 1) ? hi_bf(r[k >> 1]) : lo_bf(r[k >> 1]);
}
__device__ __forceinline__ float vec_at(const u32x4 &r, int k, const float *) { return __uint_as_float(r[k]); }

// 16 bytes of -inf
__device__ __forceinline__ u32x4 nothing(const bf16_t *) {
  return u32x4{0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u};
}
__device__ __forceinline__ u32x4 nothing(const float *) {
  return u32x4{0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u};
}

struct Span {
  int head, nv, edges;  // elements before the first boundary, whole vectors, elements outside them
};
template <typename T>
__device__ __forceinline__ Span span_of(const T *p, int V) {
  Span s;
  s.head = min(V, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
  s.nv = (V - s.head) / kVec<T>;
  s.edges = V - s.nv * kVec<T>;
  return s;
}
// index of edge element l
template <typename T>
__device__ __forceinline__ int edge_index(const Span &s, int l) {
  return l < s.head ? l : l + s.nv * kVec<T>;
}
// the thread (of GL) that holds element i
template <typename T, int GL>
__device__ __forceinline__ int owner_of(const Span &s, int i) {
  if (i < s.head) return i;
  const int j = (i - s.head) / kVec<T>;
  return j < s.nv ? j % GL : i - s.nv * kVec<T>;
}

// ---- reductions over a group ------------------------------------------------------------------------------------------
// GL <= 64: lanes of one wavefront. GL > 64: the whole workgroup, through sh [GL / 64]; two calls with the same sh need
// a barrier between them (another reduction's, for instance).
template <int GL>
__device__ __forceinline__ float group_max(float v, float *sh) {
#pragma unroll
  for (int o = (GL < 64 ? GL : 64) / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
  if constexpr (GL > 64) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < GL / 64; ++w) v = fmaxf(v, sh[w]);
  }
  return v;
}
template <int GL>
__device__ __forceinline__ float group_add(float v, float *sh) {
#pragma unroll
  for (int o = (GL < 64 ? GL : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  if constexpr (GL > 64) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < GL / 64; ++w) v += sh[w];
  }
  return v;
}
// Orders the group's accesses to shared memory and to what it has written. Within a wavefront they are in order as they
// are: the fence keeps the compiler from moving them.
template <int GL>
__device__ __forceinline__ void group_sync() {
  if constexpr (GL > 64) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- rows ---------------------------------------------------------------------------------------------------------------
// In registers: NV vectors a thread, up to GL * NV vectors. Places behind the row's end hold -inf.
template <typename T, int GL_, int NV>
struct RowRegs {
  typedef T type;
  static constexpr int GL = GL_;
  Span s;
  u32x4 v[NV];
  float edge;

  __device__ __forceinline__ void load(const T *p, int V, int lane) {
    s = span_of(p, V);
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int j = c * GL + lane;
      v[c] = j < s.nv ? stream_16(p + s.head + j * kVec<T>) : nothing(p);
    }
    edge = lane < s.edges ? load_one(p + edge_index<T>(s, lane)) : -INFINITY;
  }
  // f(value) for each element, with -inf for places behind the end
  template <typename F>
  __device__ __forceinline__ void values(F f) const {
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) f(vec_at(v[c], k, static_cast<const T *>(nullptr)));
    f(edge);
  }
  // f(index, value), with -inf for places behind the end
  template <typename F>
  __device__ __forceinline__ void each(int lane, F f) const {
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k)
        f(s.head + (c * GL + lane) * kVec<T> + k, vec_at(v[c], k, static_cast<const T *>(nullptr)));
    f(edge_index<T>(s, lane), edge);
  }
  // d[i] = f(value i), in the row's type
  template <typename F>
  __device__ __forceinline__ void write(T *d, int lane, F f) const {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int j = c * GL + lane;
      if (j < s.nv) {
        float o[kVec<T>];
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) o[k] = f(vec_at(v[c], k, static_cast<const T *>(nullptr)));
        store_row(d + s.head + j * kVec<T>, o);
      }
    }
    if (lane < s.edges) store_one(d + edge_index<T>(s, lane), f(edge));
  }
};

// Of any length: read again by each walk.
template <typename T, int GL_>
struct RowWalk {
  typedef T type;
  static constexpr int GL = GL_;
  Span s;
  const T *p;
  float edge;
  int lane;

  __device__ __forceinline__ void load(const T *row, int V, int l) {
    p = row;
    lane = l;
    s = span_of(p, V);
    edge = lane < s.edges ? load_one(p + edge_index<T>(s, lane)) : -INFINITY;
  }
  template <typename F>
  __device__ __forceinline__ void values(F f) const {
    for (int j = lane; j < s.nv; j += GL) {
      const u32x4 r = stream_16(p + s.head + static_cast<int64_t>(j) * kVec<T>);
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) f(vec_at(r, k, p));
    }
    f(edge);
  }
  template <typename F>
  __device__ __forceinline__ void each(int l, F f) const {
    for (int j = lane; j < s.nv; j += GL) {
      const u32x4 r = stream_16(p + s.head + static_cast<int64_t>(j) * kVec<T>);
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) f(s.head + j * kVec<T> + k, vec_at(r, k, p));
    }
    f(edge_index<T>(s, lane), edge);
  }
  template <typename F>
  __device__ __forceinline__ void write(T *d, int l, F f) const {
    for (int j = lane; j < s.nv; j += GL) {
      const u32x4 r = stream_16(p + s.head + static_cast<int64_t>(j) * kVec<T>);
      float o[kVec<T>];
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) o[k] = f(vec_at(r, k, p));
      store_row(d + s.head + static_cast<int64_t>(j) * kVec<T>, o);
    }
    if (lane < s.edges) store_one(d + edge_index<T>(s, lane), f(edge));
  }
};

// exp((z - top) / temperature) as a power of two: log2 e / temperature in two parts. (Rounded to one, its error has the same
// sign for every term: 1e-8 of |z - top|, which a sum over a sequence's tokens keeps. Both parts are positive: -inf stays
// -inf in their sum.)
struct ExpScale {
  float hi, lo;
  static ExpScale of(double temperature) {
    const double s = 1.4426950408889634 / temperature;
    float h = static_cast<float>(s);
    if (static_cast<double>(h) >= s) h = nextafterf(h, 0.f);
    return {h, static_cast<float>(s - static_cast<double>(h))};
  }
};
__device__ __forceinline__ float exp_of(float z, float top, ExpScale s) {
  const float t = z - top;
  return __builtin_amdgcn_exp2f(fmaf(t, s.lo, t * s.hi));
}

// Zeros where a row counts nothing.
template <typename T, int GL>
__device__ __forceinline__ void zero_row(T *d, int V, int lane) {
  const Span s = span_of(d, V);
  const float o[kVec<T>] = {};
  for (int j = lane; j < s.nv; j += GL) store_row(d + s.head + static_cast<int64_t>(j) * kVec<T>, o);
  if (lane < s.edges) store_one(d + edge_index<T>(s, lane), 0.f);
}

// log s of a sum of exponentials, off by some 3e-8 whatever its size: the exponent's part in 64 bits, the mantissa's
// (in [1 / sqrt 2, sqrt 2]) from log1p. A float log is off by half a step of the result, 5e-7 at a vocabulary of 87383.
__device__ __forceinline__ double log_of(float s) {
  int ex;
  float m = frexpf(s, &ex);
  if (m < 0.70710678f) {
    m += m;
    ex -= 1;
  }
  return static_cast<double>(ex) * 0.6931471805599453 + static_cast<double>(log1pf(m - 1.f));
}

// Threads of a workgroup that holds groups of GL.
constexpr int group_threads(int GL) { return GL < 256 ? 256 : GL; }

// The smallest register form that holds that many vectors: calls f(GL, NV), both as integral constants; NV = 0 for rows
// that are walked.
template <typename F>
inline int row_form(int64_t vectors, F f) {
#define VK_FORM(GL, NV) \
  if (vectors <= GL * NV) return f(std::integral_constant<int, GL>{}, std::integral_constant<int, NV>{})
  VK_FORM(16, 3);
  VK_FORM(16, 6);
  VK_FORM(64, 3);
  VK_FORM(64, 6);
  VK_FORM(256, 3);
  VK_FORM(256, 6);
  VK_FORM(256, 11);
  VK_FORM(512, 11);
  VK_FORM(1024, 11);
  VK_FORM(1024, 22);
#undef VK_FORM
  return f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 0>{});
}

template <typename T, int GL, int NV>
struct RowForm {
  typedef RowRegs<T, GL, NV> type;
};
template <typename T, int GL>
struct RowForm<T, GL, 0> {
  typedef RowWalk<T, GL> type;
};

}  // namespace vk
