// A row of V logits (any V, any element address) held or walked by a group of GL consecutive threads: the 16-byte vectors
// between its first and its last 16-byte boundary, vector c GL + lane with thread `lane`, and up to 14 edge elements in
// front of and behind them, one with each of the first threads. What the operators on rows of logits share
// (objectives.hip, top_logits.hip).
#pragma once

#include <float.h>
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

// Vector c GL + lane behind p, as a row's first part that is the same for a wavefront (a scalar register there), and the
// lane's 32-bit offset: no 64-bit address a vector in the vector registers.
template <int GL, typename T>
__device__ __forceinline__ const T *vector_at(const T *p, int c, int lane) {
  return reinterpret_cast<const T *>(reinterpret_cast<const char *>(p) + c * GL * 16 + static_cast<uint32_t>(lane) * 16u);
}
template <int GL, typename T>
__device__ __forceinline__ T *vector_at(T *p, int c, int lane) {
  return reinterpret_cast<T *>(reinterpret_cast<char *>(p) + c * GL * 16 + static_cast<uint32_t>(lane) * 16u);
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
template <int GL>
__device__ __forceinline__ double group_add(double v, double *sh) {
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
// At temperature 1, for log-probabilities whose small differences count: what the rounded exponent p = t log2 e leaves,
// t - p log 2, to first order behind it; 2e-7 of the exponential instead of 1e-6 for a logit 24 below the top, two operations
// an element (32 x 147 x 21847 bf16, preference: 100 -> 107 us; 16416 x 5463 bf16, policy: 72 -> 74). (-inf leaves a NaN there,
// for which med3 gives a number: times 0.)
struct UnitScale {
  static constexpr float hi = 1.4426950216293335f;
};
__device__ __forceinline__ float exp_of(float z, float top, UnitScale) {
  const float t = z - top, p = t * UnitScale::hi, e = __builtin_amdgcn_exp2f(p);
  return fmaf(e, __builtin_amdgcn_fmed3f(fmaf(p, -0.6931471806f, t), -1e-4f, 1e-4f), e);
}
// For a log-sum-exp alone: the exponential is off by 2^-24 |z - top| of itself more, all to one side, which is no more of the
// result. A thread adds those of a 16-byte vector, then the vectors, in 32 bits where it holds 22 at most and in 64 where it
// walks (a running sum in 32 rounds at its own size with every term, to the same side where terms are equal: 5e-5 of 2^22
// logits on 1024 threads, 1e-4 of 2^24. In 64 everywhere, 2064 x 87383 bf16 took 106 us instead of 100).
__device__ __forceinline__ float exp_near(float z, float top, ExpScale s) {
  return __builtin_amdgcn_exp2f((z - top) * s.hi);
}
template <typename T>
__device__ __forceinline__ float exps_near(const u32x4 &v, float top, ExpScale s) {
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kVec<T>; ++k) sum += exp_near(vec_at(v, k, static_cast<const T *>(nullptr)), top, s);
  return sum;
}

// ... of a gradient of type T: a bf16's last place is far above the scale's low part.
template <typename T, typename Scale>
__device__ __forceinline__ float exp_out(float z, float top, Scale s) {
  return sizeof(T) == 2 ? __builtin_amdgcn_exp2f((z - top) * s.hi) : exp_of(z, top, s);
}

// ---- rows ---------------------------------------------------------------------------------------------------------------
// In registers: NV vectors a thread, up to GL * NV vectors. Places behind the row's end hold -inf.
template <typename T, int GL_, int NV>
struct RowRegs {
  typedef T type;
  static constexpr bool WALKS = false;
  static constexpr int GL = GL_;
  // Exponentials stay in registers from the sum to the gradient: in the logits' place (fp32), or beside them up to 6 vectors
  // of bf16. Beyond that they are computed again.
  static constexpr bool KEEPS = sizeof(T) == 4 || NV <= 6;
  // Wavefronts a SIMD that the policy's kernel is compiled for: rows of 22 vectors a lane come out a few registers over three
  // (8192 x 11000 bf16: 82 -> 72 us); a workgroup of 1024 needs four.
  static constexpr int WAVES_A_SIMD = GL_ == 1024 ? 4 : GL_ == 64 && NV == 22 ? 3 : 1;
  // ... that the log-ratios are: 85 registers are enough (32 x 147 x 21847 bf16, 256 threads a row: 39 -> 35 us)
  static constexpr int RATIO_WAVES = GL_ == 256 || GL_ == 512 ? 6 : GL_ == 64 && NV > 3 ? 4 : 1;
  // ... that the distillation is: one register short of four
  static constexpr int DISTILL_WAVES = GL_ > 64 ? 4 : 1;
  // ... that top_logits is, and the maxima a lane of a wavefront's row that its bound comes from
  static constexpr int TOP_WAVES = GL_ > 64 ? 4 : NV <= 3 ? 8 : NV <= 6 ? 6 : NV <= 11 ? 4 : 3, TOP_MAXIMA = NV <= 6 ? NV : 4;
  Span s;
  u32x4 v[NV];
  float edge, e[sizeof(T) == 2 && KEEPS ? NV * 8 : 1];

  __device__ __forceinline__ void load(const T *p, int V, int lane) {
    s = span_of(p, V);
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int j = c * GL + lane;
      v[c] = j < s.nv ? stream_16(vector_at<GL>(p + s.head, c, lane)) : nothing(p);
    }
    // (an element of the row for every lane: a load under a branch would be waited for there)
    const float x = load_one(p + (lane < s.edges ? edge_index<T>(s, lane) : 0));
    edge = lane < s.edges ? x : -INFINITY;
  }
  // Between two walks: the vectors stay as they are. (The compiler keeps every element of the first walk unpacked for the
  // next ones otherwise, twice the registers.)
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int c = 0; c < NV; ++c) asm("" : "+v"(v[c]));
  }
  // The largest of every M-th of the thread's vectors.
  template <int M>
  __device__ __forceinline__ void maxima(float (&m)[M]) const {
#pragma unroll
    for (int i = 0; i < M; ++i) m[i] = i ? -INFINITY : edge;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) m[c % M] = fmaxf(m[c % M], vec_at(v[c], k, static_cast<const T *>(nullptr)));
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
  // Zeros for a row that counts nothing.
  static __device__ __forceinline__ void zero(T *d, int V, int lane) {
    const Span s = span_of(d, V);
    const float o[kVec<T>] = {};
#pragma unroll
    for (int c = 0; c < NV; ++c)
      if (c * GL + lane < s.nv) store_row(vector_at<GL>(d + s.head, c, lane), o);
    if (lane < s.edges) store_one(d + edge_index<T>(s, lane), 0.f);
  }
  // The thread's sum of exp((z - top) / temperature). In 64 bits: 32 round at the largest term's last place with every term
  // that follows it, 3e-7 of the sum after 88 of them, where the terms' own errors are 1e-7 of the small ones alone.
  template <typename Scale>
  __device__ __forceinline__ double exps(float top, Scale scale) {
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) {
        const float x = exp_of(vec_at(v[c], k, static_cast<const T *>(nullptr)), top, scale);
        sum += static_cast<double>(x);
        if constexpr (sizeof(T) == 4)
          v[c][k] = __float_as_uint(x);
        else if constexpr (KEEPS)
          e[c * 8 + k] = x;
      }
    const float x = exp_of(edge, top, scale);
    if constexpr (KEEPS) edge = x;
    return sum + static_cast<double>(x);
  }
  // The same for a log-sum-exp alone (exp_near).
  __device__ __forceinline__ float sum_near(float top, ExpScale scale) const {
    float sum = exp_near(edge, top, scale);
#pragma unroll
    for (int c = 0; c < NV; ++c) sum += exps_near<T>(v[c], top, scale);
    return sum;
  }
  // d[i] = factor exp((z_i - top) / temperature), in the row's type, after exps.
  template <typename Scale>
  __device__ __forceinline__ void write(T *d, int lane, float top, Scale scale, float factor) const {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int j = c * GL + lane;
      if (j < s.nv) {
        float o[kVec<T>];
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) {
          const float x = vec_at(v[c], k, static_cast<const T *>(nullptr));
          if constexpr (sizeof(T) == 2 && KEEPS)
            o[k] = e[c * 8 + k] * factor;
          else
            o[k] = (KEEPS ? x : exp_out<T>(x, top, scale)) * factor;
        }
        store_row(vector_at<GL>(d + s.head, c, lane), o);
      }
    }
    if (lane < s.edges) store_one(d + edge_index<T>(s, lane), (KEEPS ? edge : exp_of(edge, top, scale)) * factor);
  }
  // ... where another pass had the row's maximum and sum: without exps before.
  template <typename Scale>
  __device__ __forceinline__ void write_fresh(T *d, int lane, float top, Scale scale, float factor) const {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int j = c * GL + lane;
      if (j < s.nv) {
        float o[kVec<T>];
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) o[k] = exp_out<T>(vec_at(v[c], k, static_cast<const T *>(nullptr)), top, scale) * factor;
        store_row(vector_at<GL>(d + s.head, c, lane), o);
      }
    }
    if (lane < s.edges) store_one(d + edge_index<T>(s, lane), exp_of(edge, top, scale) * factor);
  }
};

// A row of up to NE elements in one thread. (Its loads and stores are 2 or 4 bytes a lane, a row's length apart; the lines
// they share stay in the caches. 512 x 1024 rows of 7 bf16 with the policy's 64-bit numbers: 16 us, 133 with 16 lanes a row;
// 131072 rows of 20: 28 and 52; of 64, lists of 32: 138 and 85. The distillation has no such form: its rows of 7 and 20 take 16
// lanes, 512 x 1024 of them 187 and 218 us.)
template <typename T, int NE>
struct RowLane {
  typedef T type;
  static constexpr int WAVES_A_SIMD = 1, RATIO_WAVES = 1, DISTILL_WAVES = 1;
  static constexpr bool WALKS = false;
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
  static __device__ __forceinline__ void zero(T *d, int V, int lane) {
    for (int k = 0; k < V; ++k) store_one(d + k, 0.f);
  }
  template <typename Scale>
  __device__ __forceinline__ double exps(float top, Scale scale) const {
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < NE; ++k) sum += exp_of(z[k], top, scale);
    return sum;
  }
  template <typename Scale>
  __device__ __forceinline__ void write(T *d, int lane, float top, Scale scale, float factor) const {
#pragma unroll
    for (int k = 0; k < NE; ++k)
      if (k < n) store_one(d + k, exp_of(z[k], top, scale) * factor);
  }
  template <typename Scale>
  __device__ __forceinline__ void write_fresh(T *d, int lane, float top, Scale scale, float factor) const {
    write(d, lane, top, scale, factor);
  }
};

// Of any length: read again by each walk.
template <typename T, int GL_>
struct RowWalk {
  typedef T type;
  static constexpr int WAVES_A_SIMD = 1, RATIO_WAVES = 1, DISTILL_WAVES = 1;
  static constexpr bool WALKS = true;
  static constexpr int GL = GL_, TOP_WAVES = 1, TOP_MAXIMA = 1;
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
  // (every thread makes every step, with -inf behind the end: f may vote)
  template <typename F>
  __device__ __forceinline__ void values(F f) const {
    for (int j0 = 0; j0 < s.nv; j0 += GL) {
      const int j = j0 + lane;
      const u32x4 r = j < s.nv ? stream_16(p + s.head + static_cast<int64_t>(j) * kVec<T>) : nothing(p);
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) f(vec_at(r, k, p));
    }
    f(edge);
  }
  template <typename F>
  __device__ __forceinline__ void each(int l, F f) const {
    for (int j0 = 0; j0 < s.nv; j0 += GL) {
      const int j = j0 + lane;
      const u32x4 r = j < s.nv ? stream_16(p + s.head + static_cast<int64_t>(j) * kVec<T>) : nothing(p);
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) f(s.head + j * kVec<T> + k, vec_at(r, k, p));
    }
    f(edge_index<T>(s, lane), edge);
  }
  static __device__ __forceinline__ void zero(T *d, int V, int lane) {
    const Span s = span_of(d, V);
    const float o[kVec<T>] = {};
    for (int j = lane; j < s.nv; j += GL) store_row(d + s.head + static_cast<int64_t>(j) * kVec<T>, o);
    if (lane < s.edges) store_one(d + edge_index<T>(s, lane), 0.f);
  }
  __device__ __forceinline__ double sum_near(float top, ExpScale scale) const {
    double sum = static_cast<double>(exp_near(edge, top, scale));
    for (int j = lane; j < s.nv; j += GL)
      sum += static_cast<double>(exps_near<T>(stream_16(p + s.head + static_cast<int64_t>(j) * kVec<T>), top, scale));
    return sum;
  }
  // Steps of a walk that are loaded together.
  static constexpr int U = 4;
  // d[i] = factor exp((z_i - top) / temperature)
  template <typename Scale>
  __device__ __forceinline__ void write_fresh(T *d, int l, float top, Scale scale, float factor) const {
    for (int j0 = 0; j0 < s.nv; j0 += GL * U) {
      u32x4 r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * GL + lane;
        r[u] = j < s.nv ? stream_16(p + s.head + static_cast<int64_t>(j) * kVec<T>) : nothing(p);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * GL + lane;
        float o[kVec<T>];
#pragma unroll
        for (int k = 0; k < kVec<T>; ++k) o[k] = exp_of(vec_at(r[u], k, p), top, scale) * factor;
        if (j < s.nv) store_row(d + s.head + static_cast<int64_t>(j) * kVec<T>, o);
      }
    }
    if (lane < s.edges) store_one(d + edge_index<T>(s, lane), exp_of(edge, top, scale) * factor);
  }
  template <typename Scale>
  __device__ __forceinline__ void write(T *d, int l, float top, Scale scale, float factor) const {
    write_fresh(d, l, top, scale, factor);
  }
};

template <int GL>
struct RowSums {  // a number a wavefront, in shared memory
  float top[GL > 64 ? GL / 64 : 1];
  double sum[GL > 64 ? GL / 64 : 1];
};
// A walked row in one pass: each thread has its own maximum so far, and its sum by that.
template <int GL, typename T, typename Scale>
__device__ __forceinline__ void walk_stats(RowWalk<T, GL> &r, Scale scale, RowSums<GL> &sh, float &top,
                                           double &s) {
  constexpr int U = RowWalk<T, GL>::U;
  float m = fmaxf(r.edge, -FLT_MAX);  // (finite: -inf - m stays -inf)
  double sum = exp_of(r.edge, m, scale);
  for (int j0 = 0; j0 < r.s.nv; j0 += GL * U) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * GL + r.lane;
      v[u] = j < r.s.nv ? stream_16(r.p + r.s.head + static_cast<int64_t>(j) * kVec<T>) : nothing(r.p);
    }
    float n = m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) n = fmaxf(n, vec_at(v[u], k, r.p));
    sum *= static_cast<double>(exp_of(m, n, scale));
    m = n;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int k = 0; k < kVec<T>; ++k) sum += static_cast<double>(exp_of(vec_at(v[u], k, r.p), m, scale));
  }
  top = group_max<GL>(m, sh.top);
  s = group_add<GL>(sum * static_cast<double>(exp_of(m, top, scale)), sh.sum);
}

// A row's maximum and its sum of exp((z - maximum) / temperature), in every thread of the group.
template <int GL, typename Row, typename Scale>
__device__ __forceinline__ void row_stats(Row &r, Scale scale, RowSums<GL> &sh, float &top, double &s) {
  if constexpr (Row::WALKS) {
    walk_stats<GL>(r, scale, sh, top, s);
    return;
  }
  top = -INFINITY;
  r.values([&](float x) { top = fmaxf(top, x); });
  top = group_max<GL>(top, sh.top);
  r.keep();
  if constexpr (!Row::WALKS) s = group_add<GL>(r.exps(top, scale), sh.sum);
  r.keep();
}
// log s, off by 1e-12: s = 2^ex m with m in [1 / sqrt 2, sqrt 2], log m = 2 atanh f, f = (m - 1) / (m + 1), |f| < 0.172.
__device__ __forceinline__ double log_of(double s) {
  int ex;
  double m = frexp(s, &ex);
  if (m < 0.70710678) {
    m += m;
    ex -= 1;
  }
  const double f = (m - 1.0) / (m + 1.0), g = f * f;
  double t = 1.0 / 15.0;
#pragma unroll
  for (int n = 13; n >= 1; n -= 2) t = fma(t, g, 1.0 / n);
  t = fma(static_cast<double>(ex), 0.6931471805599453, 2.0 * f * t);
  return s > 0.0 ? t : s == 0.0 ? -INFINITY : s;  // (NaN stays)
}
// The same as a call, beside a row that fills the registers: the constants of the series stay out of them
// (2064 x 87383 fp32, distillation: 300 us inlined, 285 called; 32 x 147 x 21847 bf16, preference: 111 and 107). Not all of them:
// rows of 1024 threads of 22 vectors still have 44 (bf16) and 46 (fp32) registers in memory there, and 22 to 44 in the
// policy's kernel, which has the logarithm inlined.
static __device__ __attribute__((noinline)) double log_called(double s) { return log_of(s); }

// The same of a sum in 32 bits, off by 3e-8 whatever its size: the exponent's part in 64 bits, the mantissa's from log1p.
__device__ __forceinline__ double log_near(float s) {
  int ex;
  float m = frexpf(s, &ex);
  if (m < 0.70710678f) {
    m += m;
    ex -= 1;
  }
  return static_cast<double>(ex) * 0.6931471805599453 + static_cast<double>(log1pf(m - 1.f));
}

// exp(x) - 1 - x for |x| < 1/2, off by 1e-10 of it: nine terms.
__device__ __forceinline__ double series_beyond_line(double x) {
  double t = 1.0;
#pragma unroll
  for (int n = 11; n >= 3; --n) t = fma(t * x, 1.0 / n, 1.0);
  return 0.5 * x * x * t;
}
// exp(x) - 1 - x beyond: x halved until it is under 1/2, then expm1(2 y) = expm1(y) (expm1(y) + 2). A call: few tokens need
// it, and its registers would be taken from every row.
static __device__ __attribute__((noinline)) double exp_far_beyond_line(double x) {
  int m;
  frexp(x, &m);
  const bool huge = !(fabs(x) <= 800.0);
  if (huge) return x > 0.0 ? INFINITY : x < 0.0 ? -1.0 - x : x;
  const double y = ldexp(x, -(m + 1));
  double e = y + series_beyond_line(y);
  for (; m >= 0; --m) e *= e + 2.0;
  return e - x;
}
// exp(x) for |x| >= 1/2: halved likewise, then squared (off by 1e-10 of it at 10, 1e-8 at 700).
static __device__ __attribute__((noinline)) double exp_far(double x) {
  int m;
  frexp(x, &m);
  if (!(fabs(x) <= 800.0)) return x > 0.0 ? INFINITY : x < 0.0 ? 0.0 : x;
  const double y = ldexp(x, -(m + 1));
  double e = 1.0 + (y + series_beyond_line(y));
  for (; m >= 0; --m) e *= e;
  return e;
}
// exp(x) - 1 - x without cancellation
__device__ __forceinline__ double exp_beyond_line(double x) {
  return fabs(x) < 0.5 ? series_beyond_line(x) : exp_far_beyond_line(x);
}
__device__ __forceinline__ double exp_64(double x) {
  return fabs(x) < 0.5 ? 1.0 + (x + series_beyond_line(x)) : exp_far(x);
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

// The smallest register form of at least 16 lanes that holds that many vectors: calls f(GL, NV), both as integral constants;
// NV = 0 for rows that are walked. A wavefront a row (no barriers) as far as its registers go: 16416 x 5463 bf16, policy and
// distillation, 71 and 91 us with 64 lanes of 11 vectors, 84 and 111 with 256 of 3, 116 and 185 with 512 of 2; beyond 22
// vectors a lane it loses (4704 x 21847 bf16, preference: 108 us with 64 lanes of 43, 100 with 256 of 11). 16 lanes where four
// rows to a wavefront share the 64-bit numbers: 131072 x 343 fp32, policy, 83 us with 16 lanes of 6, 144 with 64 of 2; the
// other way round from 100 vectors on (112500 x 800 bf16: 153 and 128). Rows past 22528 vectors are read twice: 2064 x 87383 fp32,
// distillation, 390 us walked, 288 in registers; of 90112 and 90300 logits, 289 and 411.
// A row pays the exponentials of all the vectors of its form, so that one just past a form's end costs more than its bytes:
// policy, 16416 rows of 5632 and 5640 bf16 75 and 98 us, 4704 of 11264 and 11300 51 and 65.
template <typename F>
inline int row_form(int64_t vectors, F f) {
#define VK_FORM(GL, NV) \
  if (vectors <= GL * NV) return f(std::integral_constant<int, GL>{}, std::integral_constant<int, NV>{})
  VK_FORM(16, 3);
  VK_FORM(16, 6);
  VK_FORM(64, 2);
  VK_FORM(64, 3);
  VK_FORM(64, 6);
  VK_FORM(64, 11);
  VK_FORM(64, 22);
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
