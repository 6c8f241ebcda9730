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
  if constexpr (GL == 1) return 0;
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
  // Between two walks: the vectors stay as they are. (The compiler keeps every element of the first walk unpacked for the
  // next ones otherwise, twice the registers.)
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int c = 0; c < NV; ++c) asm("" : "+v"(v[c]));
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

// A row of up to NE elements in one thread. (Its loads and stores are 2 or 4 bytes a lane, a row's length apart; the lines
// they share stay in the caches: 512 x 1024 rows of 7 bf16 move 4.9 TB/s so.)
template <typename T, int NE>
struct RowLane {
  typedef T type;
  static constexpr int GL = 1;
  Span s;
  float z[NE];
  int n;

  __device__ __forceinline__ void load(const T *p, int V, int lane) {
    n = V;
#pragma unroll
    for (int k = 0; k < NE; ++k) z[k] = k < V ? load_one(p + k) : -INFINITY;
  }
  __device__ __forceinline__ void keep() {}
  template <typename F>
  __device__ __forceinline__ void values(F f) const {
#pragma unroll
    for (int k = 0; k < NE; ++k) f(z[k]);
  }
  template <typename F>
  __device__ __forceinline__ void write(T *d, int lane, F f) const {
#pragma unroll
    for (int k = 0; k < NE; ++k)
      if (k < n) store_one(d + k, f(z[k]));
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
  __device__ __forceinline__ void keep() {}
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
  for (int l = lane; l < s.edges; l += GL) store_one(d + edge_index<T>(s, l), 0.f);
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

// exp(x) - 1, off by a few 1e-16 of it (and of x near 0): a series on x halved until it is under 1/2, then
// expm1(2 y) = expm1(y) (expm1(y) + 2). A dozen registers, where the library's takes thirty from the row.
__device__ __forceinline__ double series_beyond_line(double x) {  // exp(x) - 1 - x for |x| < 1/2
  double t = 1.0;
#pragma unroll
  for (int n = 14; n >= 3; --n) t = fma(t * x, 1.0 / n, 1.0);
  return 0.5 * x * x * t;
}
__device__ __forceinline__ double expm1_of(double x) {
  int m;
  frexp(x, &m);
  if (!(fabs(x) >= 0.5) || fabs(x) > 800.0) m = -1;
  const double y = ldexp(fabs(x) > 800.0 ? 0.0 : x, -(m + 1));
  double e = y + series_beyond_line(y);
  for (; m >= 0; --m) e *= e + 2.0;
  if (x > 800.0) e = INFINITY;
  if (x < -800.0) e = -1.0;
  return e;
}
// exp(x) - 1 - x without cancellation
__device__ __forceinline__ double exp_beyond_line(double x) {
  return fabs(x) < 0.5 ? series_beyond_line(x) : expm1_of(x) - x;
}

// Threads of a workgroup that holds groups of GL; a thread's group, known to be the same for a wavefront where it is (row
// numbers and row addresses are scalars then); its place in the group.
constexpr int group_threads(int GL) { return GL < 256 ? 256 : GL; }
template <int GL>
__device__ __forceinline__ int group_of() {
  if constexpr (GL >= 256) return 0;
  if constexpr (GL >= 64) return __builtin_amdgcn_readfirstlane(threadIdx.x / GL);
  return threadIdx.x / GL;
}
template <int GL>
__device__ __forceinline__ int lane_of() {
  if constexpr (GL >= 256) return threadIdx.x;
  return threadIdx.x % GL;
}

// The smallest register form of at least 16 lanes that holds that many vectors: calls f(GL, NV), both as integral constants; NV = 0 for rows
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

// GL = 1: NV is the number of elements
template <typename T, int GL, int NV>
struct RowForm {
  typedef RowRegs<T, GL, NV> type;
};
template <typename T, int GL>
struct RowForm<T, GL, 0> {
  typedef RowWalk<T, GL> type;
};
template <typename T, int NE>
struct RowForm<T, 1, NE> {
  typedef RowLane<T, NE> type;
};

}  // namespace vk
