// Rules on logits and the token choice at any vocabulary (select.hip: the fused LM head + choice up to 512 tokens).
//
// Rules, for sequence b and token v with x = logits[b, v] in fp32 and c = how often v occurs in b's history:
//   c > 0:  z = x > 0 ? x / repetition_b : x * repetition_b;  z -= frequency_b * c;  z -= presence_b
//   z += bias[v];  v not allowed: z = -inf whatever it was (a NaN or an infinity in a masked place is not read into)
// every step rounded to fp32 in this order and none contracted, so the result is the one of the elementary operations.
// Choice: z' = z / T (T > 0); greedy: the first index of max z; Gumbel: the first index of max z' - log(-log max(u, 1e-20))
// with one uniform per (sequence, token); inverse CDF: the first index whose running softmax(z') sum exceeds u. A NaN is
// never chosen and weighs nothing; +inf counts as the largest finite value. log-probability: z' of the choice minus
// log sum exp z'. A row with nothing left takes the fallback token, log-probability -inf.
//
// A workgroup takes one slice of one sequence's vocabulary and counts the history's tokens of that slice in LDS (16 bits
// each), so no count per (sequence, token) exists in memory. Slices give (max, sum of exponentials at it, best); one
// wavefront per sequence joins them.
#include <float.h>
#include <math.h>

#include "decode_state.h"
#include "row_access.h"

namespace vk {

constexpr int CH_THREADS = 256;
constexpr int CH_SLICE = 16384;   // tokens of a slice at most: 32 KB of LDS counts
constexpr int CH_SLICE_MIN = 2048;
constexpr int CH_HIST_MAX = 65535;  // a count has 16 bits

struct Rules {
  const int64_t *hist;  // [B, hist_cols], row stride hist_ld; null: no penalties
  int64_t hist_ld, hist_cols;
  const int32_t *len;   // [B]; null: pos - plen
  const int64_t *pos, *plen;
  const float *rep, *pres, *freq;  // [B] or null: the scalar
  float rep0, pres0, freq0;
  const float *bias;  // row b at b * bias_ld; null: none
  int64_t bias_ld;
  const uint32_t *allowed;  // [n_allowed, allowed_ld] bit masks; null: none
  int64_t allowed_ld, n_allowed;
  const int32_t *arow;       // [B] mask row, outside 0 .. n_allowed - 1: no mask
  const int32_t *token_row;  // [V] mask row by previous token (with tok)
  const int64_t *tok;
};

struct RowRules {
  const int64_t *hist;
  int len;  // 0: no penalties
  float rep, pres, freq;
  const float *bias;
  const uint32_t *allowed;
};

__device__ __forceinline__ RowRules row_rules(const Rules &r, int64_t b, int V) {
  RowRules o = {};
  if (r.hist != nullptr) {
    o.rep = r.rep ? r.rep[b] : r.rep0;
    o.pres = r.pres ? r.pres[b] : r.pres0;
    o.freq = r.freq ? r.freq[b] : r.freq0;
    int64_t n = r.len ? r.len[b] : r.pos[b] - (r.plen ? r.plen[b] : 0);
    n = n < 0 ? 0 : (n > r.hist_cols ? r.hist_cols : n);
    o.hist = r.hist + b * r.hist_ld;
    // repetition 1 divides and multiplies by one, and the others subtract zero: nothing to count
    o.len = o.rep == 1.f && o.pres == 0.f && o.freq == 0.f ? 0 : static_cast<int>(n);
  }
  o.bias = r.bias ? r.bias + b * r.bias_ld : nullptr;
  if (r.allowed != nullptr) {
    int64_t a = b;
    if (r.token_row != nullptr) {
      const int64_t t = r.tok[b];
      a = t >= 0 && t < V ? r.token_row[t] : -1;
    } else if (r.arow != nullptr) {
      a = r.arow[b];
    } else if (r.n_allowed == 1) {
      a = 0;
    }
    if (a >= 0 && a < r.n_allowed) o.allowed = r.allowed + a * r.allowed_ld;
  }
  return o;
}

// cnt: 16-bit counts, two a word, of tokens v0 .. v0 + slice - 1 in hist[0 .. len - 1] (slice % 32 == 0). Ends with a
// barrier.
__device__ __forceinline__ void count_history(uint32_t *cnt, const int64_t *hist, int len, int v0, int slice) {
  const int64_t first = hist[threadIdx.x < len ? threadIdx.x : 0];  // in flight while the counts are cleared
  for (int i = threadIdx.x; i < slice / 8; i += CH_THREADS) reinterpret_cast<u32x4 *>(cnt)[i] = u32x4{0u, 0u, 0u, 0u};
  __syncthreads();
  for (int t = threadIdx.x; t < len; t += CH_THREADS) {
    const int64_t rel = (t == static_cast<int>(threadIdx.x) ? first : hist[t]) - v0;
    if (rel >= 0 && rel < slice) atomicAdd(&cnt[rel >> 1], (rel & 1) ? 0x10000u : 1u);
  }
  __syncthreads();
}

// N consecutive tokens' logits and what the rules read for them, loaded ahead of their use. A vector that does not fit
// into the row (its last one, where N does not divide V) is read one by one when it is used; its place here holds the
// row's last whole vector, so that every load is unconditional and in bounds.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  u32x4 raw;
  float bias[N];
  uint32_t mask;

  __device__ __forceinline__ void load(const T *row, const RowRules &r, int v, int V) {
    if (V < N) return;
    const int at = v <= V - N ? v : V - N;
    raw = load_16(row + at);
    if (r.bias != nullptr) load_row<N>(r.bias + at, bias);
    if (r.allowed != nullptr) mask = r.allowed[at >> 5];
  }

  // z: the logits after the rules, -inf past the row's end. v < V, v % N == 0; cnt: the counts of tokens v, v + 1, ...
  __device__ __forceinline__ void rules(float (&z)[N], const T *row, const RowRules &r, const uint32_t *cnt, int v, int V) {
#pragma clang fp contract(off)
    const bool whole = v <= V - N;
    if (whole) {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if constexpr (sizeof(T) == 4)
          z[k] = __uint_as_float(raw[k]);
        else
          z[k] = (k & 1) ? hi_bf(raw[k / 2]) : lo_bf(raw[k / 2]);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = load_one(row + (v + k < V ? v + k : V - 1));
      if (r.bias != nullptr)
#pragma unroll
        for (int k = 0; k < N; ++k) bias[k] = r.bias[v + k < V ? v + k : V - 1];
      if (r.allowed != nullptr) mask = r.allowed[v >> 5];
    }
    if (r.len > 0) {
      uint32_t w[N / 2], any = 0;
#pragma unroll
      for (int k = 0; k < N / 2; ++k) any |= w[k] = cnt[k];
      if (any) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int c = (k & 1) ? w[k / 2] >> 16 : w[k / 2] & 0xffff;
          if (c > 0) {
            z[k] = z[k] > 0.f ? z[k] / r.rep : z[k] * r.rep;
            z[k] = z[k] - r.freq * static_cast<float>(c);
            z[k] = z[k] - r.pres;
          }
        }
      }
    }
    if (r.bias != nullptr)
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = z[k] + bias[k];
    if (r.allowed != nullptr) {
      const uint32_t bits = mask >> (v & 31);
#pragma unroll
      for (int k = 0; k < N; ++k) z[k] = (bits >> k) & 1 ? z[k] : -INFINITY;
    }
    if (!whole)
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (v + k >= V) z[k] = -INFINITY;
  }
};

// Vectors that a thread has in flight: 16 elements.
template <typename T>
constexpr int kAhead = sizeof(T);

// grid: B x slices workgroups, a sequence's slices side by side. out may be logits.
template <typename T, typename OT>
__global__ __launch_bounds__(CH_THREADS) void process_logits_kernel(const T *logits, int64_t ld, Rules rules, int V,
                                                                    int slices, int slice, OT *out, int64_t out_ld) {
  extern __shared__ __attribute__((aligned(16))) uint32_t cnt[];
  constexpr int N = Vec<T>::N, R = kAhead<T>, STEP = CH_THREADS * N;
  const int64_t b = blockIdx.x / slices;
  const int v0 = static_cast<int>(blockIdx.x % slices) * slice, v1 = V - v0 < slice ? V : v0 + slice;
  const RowRules r = row_rules(rules, b, V);
  const T *row = logits + b * ld;
  OT *dst = out + b * out_ld;
  const int mine = v0 + static_cast<int>(threadIdx.x) * N;
  Vec<T> x[R];
  for (int w = v0; w < v1; w += R * STEP) {
#pragma unroll
    for (int q = 0; q < R; ++q) x[q].load(row, r, w - v0 + mine + q * STEP, V);
    if (w == v0 && r.len > 0) count_history(cnt, r.hist, r.len, v0, slice);
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int v = w - v0 + mine + q * STEP;
      if (v >= v1) continue;
      float z[N];
      x[q].rules(z, row, r, cnt + (v - v0) / 2, v, V);
      if (v <= V - N) {
        store_row<N>(dst + v, z);
      } else {
        for (int k = 0; k < N && v + k < V; ++k) store_one(dst + v + k, z[k]);
      }
    }
  }
}

// ---- the choice --------------------------------------------------------------------------------------------------------

enum { CH_GREEDY = 0, CH_GUMBEL = 1, CH_CDF = 2 };

// Running state of a part of a row: the maximum of z (at least -FLT_MAX), the sum of exp((z - m) / T), and the best token.
// Gumbel: v is that token, s its score in fp32 (within score_slack of the exact one), z its logit and u its uniform.
// Else: z is the largest logit (-inf: none) and v the first token, or the first token of the vector, that has it.
struct Part {
  float m, sum, s, z, u;
  int32_t v;  // -1: none yet
};

__device__ __forceinline__ Part no_part() { return {-FLT_MAX, 0.f, -INFINITY, -INFINITY, 0.f, -1}; }

// How far the fp32 score of a token can be from the exact one: the roundings of z' and of the sum (1.2e-7 of its size
// each), and of the two logarithms.
__device__ __forceinline__ float score_slack(float s) { return 1e-5f + 1e-6f * fabsf(s); }

// The exact score: z' rounded to fp32, the noise in 64 bits.
__device__ __forceinline__ double exact_score(float z, float u, float T) {
  return static_cast<double>(z / T) - log(-log(fmax(static_cast<double>(u), 1e-20)));
}

// Whether b's token comes before a's. Gumbel scores that fp32 cannot order are compared in 64 bits.
template <bool GUMBEL>
__device__ __forceinline__ bool better(const Part &a, const Part &b, float T) {
  if (b.v < 0) return false;
  if (a.v < 0) return true;
  if (GUMBEL && T > 0.f) {
    const float d = b.s - a.s;
    if (fabsf(d) > 2.f * score_slack(fmaxf(fabsf(a.s), fabsf(b.s)))) return d > 0.f;
    const double ea = exact_score(a.z, a.u, T), eb = exact_score(b.z, b.u, T);
    return eb > ea || (eb == ea && b.v < a.v);
  }
  return b.z > a.z || (b.z == a.z && b.v < a.v);
}

// L: log2(e) / T. Differences first: nothing overflows where all logits are the type's lowest value.
template <bool GUMBEL>
__device__ __forceinline__ void join_parts(Part &a, const Part &b, float L, float T) {
  const float M = fmaxf(a.m, b.m);
  a.sum = a.sum * __builtin_amdgcn_exp2f((a.m - M) * L) + b.sum * __builtin_amdgcn_exp2f((b.m - M) * L);
  a.m = M;
  if (better<GUMBEL>(a, b, T)) {
    a.s = b.s;
    a.z = b.z;
    a.u = b.u;
    a.v = b.v;
  }
}

template <bool GUMBEL>
__device__ __forceinline__ void join_lanes(Part &p, float L, float T) {
#pragma unroll 1
  for (int o = 32; o > 0; o >>= 1) {
    Part q;
    q.m = __shfl_xor(p.m, o, 64);
    q.sum = __shfl_xor(p.sum, o, 64);
    q.s = GUMBEL ? __shfl_xor(p.s, o, 64) : 0.f;
    q.z = __shfl_xor(p.z, o, 64);
    q.u = GUMBEL ? __shfl_xor(p.u, o, 64) : 0.f;
    q.v = __shfl_xor(p.v, o, 64);
    join_parts<GUMBEL>(p, q, L, T);
  }
}

// A NaN becomes -inf, +inf the largest finite value: v_med3_f32 of a NaN is the smaller of the others. As asm: the
// compiler's own med3 with -inf is a minimum, which a NaN passes as the other operand.
__device__ __forceinline__ float tame(float z) {
  float d;
  asm("v_med3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(z), "v"(-INFINITY), "v"(FLT_MAX));
  return d;
}

struct Scale {
  float T, inv, L;  // the temperature, 1 / T (1 for a greedy row) kept finite, and log2(e) / T
};

__device__ __forceinline__ Scale row_scale(const float *temp, float temp0, int64_t b) {
  Scale c;
  c.T = temp ? temp[b] : temp0;
  c.inv = c.T > 0.f ? fminf(1.f / c.T, 0.5f * FLT_MAX) : 1.f;
  c.L = fminf(c.inv * 1.44269504f, 0.5f * FLT_MAX);
  return c;
}

// The uniforms of sequence b are at u + b * ld; in a decode step those of its output column (clamped to the columns there
// are), a column being 1 uniform (inverse CDF) or V of them (Gumbel).
struct Noise {
  const float *u;
  int64_t ld, cols;
};

__device__ __forceinline__ const float *noise_at(const Noise &n, const Rules &r, int64_t b, int64_t per_column) {
  int64_t col = 0;
  if (r.pos != nullptr) {
    col = r.pos[b] - (r.plen ? r.plen[b] : 0);
    col = col < 0 ? 0 : (col >= n.cols ? n.cols - 1 : col);
  }
  return n.u + b * n.ld + col * per_column;
}

struct Choice {
  int64_t *token;  // [B], or null with a state
  float *logp;     // [B] (logp_stride 0), or [B, columns] by output column; null: none
  int64_t logp_stride, fallback;
};

// The optional state of a decode step: tail / homo flags per token, and what advance_state needs besides.
struct Step {
  DecodeState s;
  const uint8_t *is_tail, *is_homo;
  const int64_t *plen, *rope_off;
};

__device__ __forceinline__ void finish_row(const Choice &c, const Step &st, int64_t b, int V, int64_t v, float logp) {
  if (v < 0) {
    v = c.fallback;
    logp = -INFINITY;
  }
  if (c.token) c.token[b] = v;
  int64_t p = 0, ocol = 0;
  if (st.s.pos) {
    p = st.s.pos[b];
    ocol = p - (st.plen ? st.plen[b] : 0);
  }
  if (c.logp) {
    if (c.logp_stride == 0)
      c.logp[b] = logp;
    else if (ocol >= 0 && ocol < st.s.out_cols)
      c.logp[b * c.logp_stride + ocol] = logp;
  }
  if (!st.s.pos) return;
  const int64_t prev = st.s.tok[b];
  const bool tail = prev >= 0 && prev < V && st.is_tail[prev];
  advance_state(st.s, b, v, prev, tail, st.is_homo, V, p, st.s.run ? st.s.run[b] : 0, ocol,
                st.rope_off ? st.rope_off[b] : 0, st.s.cache_base ? st.s.cache_base[b] : 0);
}

// log softmax(z')[token] of a logit z of the row that p sums.
__device__ __forceinline__ float logp_of(float z, const Part &p, const Scale &c) {
  const float d = z - p.m;
  return (c.T > 0.f ? d / c.T : d) - logf(p.sum);
}

// One slice of one sequence, or with ONE the whole vocabulary and the step's end.
template <typename T, bool GUMBEL, bool ONE>
__global__ __launch_bounds__(CH_THREADS) void choose_slices_kernel(const T *__restrict__ logits, int64_t ld, Rules rules,
                                                                   const float *__restrict__ temp, float temp0,
                                                                   Noise noise, int V, int slices, int slice,
                                                                   Part *__restrict__ parts, Choice choice, Step step) {
  extern __shared__ __attribute__((aligned(16))) uint32_t cnt[];
  __shared__ Part red[CH_THREADS / 64];
  constexpr int N = Vec<T>::N, R = kAhead<T>, STEP = CH_THREADS * N;
  const int64_t b = ONE ? blockIdx.x : blockIdx.x / slices;
  const int v0 = ONE ? 0 : static_cast<int>(blockIdx.x % slices) * slice, v1 = V - v0 < slice ? V : v0 + slice;
  const RowRules r = row_rules(rules, b, V);
  const Scale c = row_scale(temp, temp0, b);
  const bool noisy = GUMBEL && c.T > 0.f;
  const T *row = logits + b * ld;
  const float *urow = noisy ? noise_at(noise, rules, b, V) : nullptr;
  const int mine = v0 + static_cast<int>(threadIdx.x) * N;
  Part p = no_part();
  Vec<T> x[R];
  float u[GUMBEL ? R : 1][N];
  for (int w = v0; w < v1; w += R * STEP) {
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int v = w - v0 + mine + q * STEP;
      x[q].load(row, r, v, V);
      if (noisy && V >= N) load_row<N>(urow + (v <= V - N ? v : V - N), u[GUMBEL ? q : 0]);
    }
    if (w == v0 && r.len > 0) count_history(cnt, r.hist, r.len, v0, slice);
    float z[R][N], top = -INFINITY;
    int topv = -1;
#pragma unroll
    for (int q = 0; q < R; ++q) {
      const int v = w - v0 + mine + q * STEP;
      if (v < v1) {
        x[q].rules(z[q], row, r, cnt + (v - v0) / 2, v, V);
        if (noisy && v > V - N)
#pragma unroll
          for (int k = 0; k < N; ++k) u[GUMBEL ? q : 0][k] = urow[v + k < V ? v + k : V - 1];
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) z[q][k] = -INFINITY;
      }
      float most = -INFINITY;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        z[q][k] = tame(z[q][k]);
        most = vmax2(most, z[q][k]);
      }
      if (most > top) {
        top = most;
        topv = v;
      }
    }
    const float m = vmax2(p.m, top);
    p.sum *= __builtin_amdgcn_exp2f((p.m - m) * c.L);
    p.m = m;
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int k = 0; k < N; ++k) p.sum += __builtin_amdgcn_exp2f((z[q][k] - m) * c.L);
    if (!noisy) {
      if (top > p.z) {
        p.z = top;
        p.v = topv;
      }
    } else {
#pragma unroll
      for (int q = 0; q < R; ++q)
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const float uk = u[GUMBEL ? q : 0][k];
          Part t = p;
          t.z = z[q][k];
          t.u = uk;
          t.s = fmaf(t.z, c.inv, -logf(-logf(fmaxf(uk, 1e-20f))));
          t.v = t.z == -INFINITY ? -1 : w - v0 + mine + q * STEP + k;
          if (better<GUMBEL>(p, t, c.T)) p = t;
        }
    }
  }
  join_lanes<GUMBEL>(p, c.L, c.T);
  const int lane = threadIdx.x & 63;
  if (lane == 0) red[threadIdx.x >> 6] = p;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int w = 1; w < CH_THREADS / 64; ++w) join_parts<GUMBEL>(p, red[w], c.L, c.T);
  if (!noisy && p.v >= 0) {  // the token inside its vector
    float z[N];
    x[0].load(row, r, p.v, V);
    x[0].rules(z, row, r, cnt + (p.v - v0) / 2, p.v, V);
    int k = 0;
#pragma unroll
    for (int e = N - 1; e >= 0; --e) k = tame(z[e]) == p.z ? e : k;
    p.v += k;
  }
  if constexpr (ONE)
    finish_row(choice, step, b, V, p.v, logp_of(p.z, p, c));
  else
    parts[blockIdx.x] = p;
}

// One wavefront per sequence joins its slices.
template <bool GUMBEL>
__global__ __launch_bounds__(256) void choose_join_kernel(const Part *__restrict__ parts, const float *__restrict__ temp,
                                                          float temp0, int64_t B, int V, int slices, Choice choice,
                                                          Step step) {
  const int64_t b = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (b >= B) return;
  const int lane = threadIdx.x & 63;
  const Scale c = row_scale(temp, temp0, b);
  Part p = no_part();
  for (int s = lane; s < slices; s += 64) join_parts<GUMBEL>(p, parts[b * slices + s], c.L, c.T);
  join_lanes<GUMBEL>(p, c.L, c.T);
  if (lane == 0) finish_row(choice, step, b, V, p.v, logp_of(p.z, p, c));
}

// Inverse CDF: one workgroup per sequence finds the slice that u falls into from the slices' sums (64 bits), then walks
// that slice in token order, CH_THREADS x N tokens a round. A row with temperature <= 0 takes the greedy choice.
template <typename T>
__global__ __launch_bounds__(CH_THREADS) void choose_cdf_kernel(const T *__restrict__ logits, int64_t ld, Rules rules,
                                                                const float *__restrict__ temp, float temp0,
                                                                Noise noise, int V, int slices, int slice,
                                                                const Part *__restrict__ parts,
                                                                Choice choice, Step step) {
  extern __shared__ __attribute__((aligned(16))) uint32_t cnt[];
  __shared__ double wave_total[CH_THREADS / 64];
  __shared__ int found, last;
  constexpr int N = Vec<T>::N;
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const Scale c = row_scale(temp, temp0, b);
  const Part *mine = parts + b * slices;
  // every thread joins the slices the same way
  Part p = no_part();
  for (int s = 0; s < slices; ++s) join_parts<false>(p, mine[s], c.L, c.T);
  if (p.v < 0 || !(c.T > 0.f)) {
    if (tid == 0) finish_row(choice, step, b, V, p.v, logp_of(p.z, p, c));
    return;
  }
  auto weight = [&](int s) { return static_cast<double>(mine[s].sum * __builtin_amdgcn_exp2f((mine[s].m - p.m) * c.L)); };
  double total = 0.;
  for (int s = 0; s < slices; ++s) total += weight(s);
  const double target = static_cast<double>(*noise_at(noise, rules, b, 1)) * total;
  // the slice: the first whose running sum passes the target (rounding, or a uniform of 1: the last with any weight)
  int at = -1, filled = 0;
  double before = 0., run = 0.;
  for (int s = 0; s < slices && at < 0; ++s) {
    const double w = weight(s);
    if (w > 0.) {
      filled = s;
      run = before;
      if (target < before + w) at = s;
    }
    before += w;
  }
  if (at < 0) at = filled;
  const RowRules r = row_rules(rules, b, V);
  const int v0 = at * slice, v1 = V - v0 < slice ? V : v0 + slice;
  if (tid == 0) {
    found = 0x7fffffff;
    last = -1;
  }
  __syncthreads();
  if (r.len > 0) count_history(cnt, r.hist, r.len, v0, slice);
  const T *row = logits + b * ld;
  Vec<T> x;
  float z[N];
  for (int w0 = v0; w0 < v1; w0 += CH_THREADS * N) {
    const int v = w0 + tid * N;
    double e[N], sum = 0.;
    int top = -1;
#pragma unroll
    for (int k = 0; k < N; ++k) e[k] = 0.;
    if (v < v1) {
      x.load(row, r, v, V);
      x.rules(z, row, r, cnt + (v - v0) / 2, v, V);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        e[k] = static_cast<double>(__builtin_amdgcn_exp2f((tame(z[k]) - p.m) * c.L));
        if (e[k] > 0.) top = v + k;
        sum += e[k];
      }
    }
    double inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(inc, o, 64);
      if (lane >= o) inc += up;
    }
    if (lane == 63) wave_total[wid] = inc;
    __syncthreads();
    double cdf = run;
    for (int w = 0; w < CH_THREADS / 64; ++w) {
      if (w < wid) cdf += wave_total[w];
      run += wave_total[w];
    }
    cdf += inc - sum;
    int hit = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      cdf += e[k];
      if (hit == 0x7fffffff && e[k] > 0. && target < cdf) hit = v + k;
    }
    if (hit != 0x7fffffff) atomicMin(&found, hit);
    if (top >= 0) atomicMax(&last, top);
    __syncthreads();
    if (found != 0x7fffffff) break;
  }
  if (tid != 0) return;
  const int pick = found != 0x7fffffff ? found : last, v = pick & ~(N - 1);
  if (pick < 0) {  // (a slice with weight holds a token with weight)
    finish_row(choice, step, b, V, p.v, logp_of(p.z, p, c));
    return;
  }
  x.load(row, r, v, V);  // the choice's own logit again
  x.rules(z, row, r, cnt + (v - v0) / 2, v, V);
  float zt = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) zt = v + k == pick ? tame(z[k]) : zt;
  finish_row(choice, step, b, V, pick, logp_of(zt, p, c));
}

// Slices per sequence: about two workgroups per CU in all, of 2048 to 16384 tokens each.
static void slice_plan(int64_t B, int V, int *slices, int *slice) {
  const int64_t want = (2 * device_cus_cached() + B - 1) / B;
  int64_t s = (V + CH_SLICE_MIN - 1) / CH_SLICE_MIN;
  if (s > want) s = want;
  const int64_t least = (V + CH_SLICE - 1) / CH_SLICE;
  if (s < least) s = least;
  const int64_t len = ((V + s - 1) / s + 31) / 32 * 32;
  *slice = static_cast<int>(len);
  *slices = static_cast<int>((V + len - 1) / len);
}

static int check_rules(const Rules &r, int64_t B, int V, const char *what) {
  VK_CHECK_ARG(r.hist == nullptr || (r.len != nullptr || r.pos != nullptr), "%s: a history needs lengths", what);
  VK_CHECK_ARG(r.hist == nullptr || (r.hist_cols >= 0 && r.hist_cols <= CH_HIST_MAX && r.hist_ld >= r.hist_cols),
               "%s: histories of at most %d tokens", what, CH_HIST_MAX);
  VK_CHECK_ARG(r.hist == nullptr || r.rep != nullptr || r.rep0 > 0.f, "%s: the repetition penalty must be positive", what);
  VK_CHECK_ARG(r.bias == nullptr || r.bias_ld == 0 || r.bias_ld >= V, "%s: bias row stride below V", what);
  VK_CHECK_ARG(r.allowed == nullptr || (r.n_allowed > 0 && r.allowed_ld >= (V + 31) / 32),
               "%s: masks are rows of ceil(V / 32) words", what);
  VK_CHECK_ARG(r.allowed == nullptr || r.arow != nullptr || r.token_row != nullptr || r.n_allowed == 1 || r.n_allowed == B,
               "%s: masks without row numbers: 1 row or one per sequence", what);
  return VK_OK;
}

static int check_logits(const void *logits, int32_t dtype, int64_t ld, int64_t B, int32_t V, const char *what) {
  VK_CHECK_ARG(B >= 0 && V > 0 && V <= (int32_t(1) << 30) && ld >= V, "%s: bad sizes", what);
  VK_CHECK_ARG(B < (int64_t(1) << 20), "%s: at most 2^20 - 1 sequences", what);
  VK_CHECK_ARG(dtype == VK_DTYPE_BF16 || dtype == VK_DTYPE_F32, "%s: logits bf16 or fp32", what);
  VK_CHECK_ARG(B == 0 || logits != nullptr, "%s: null pointer", what);
  return VK_OK;
}

template <typename T>
static int launch_choose(const void *logits, int64_t ld, const Rules &r, const float *temp, float temp0, int mode,
                         const Noise &noise, int64_t B, int V, Part *parts, const Choice &choice, const Step &step,
                         hipStream_t s) {
  int slices, slice;
  slice_plan(B, V, &slices, &slice);
  const T *x = static_cast<const T *>(logits);
  const size_t lds = r.hist ? static_cast<size_t>(slice) * 2 : 0;
  const unsigned grid = static_cast<unsigned>(B * slices), join = static_cast<unsigned>((B + 3) / 4);
#define VK_SLICES(GUMBEL, ONE)                                                                                          \
  choose_slices_kernel<T, GUMBEL, ONE><<<grid, CH_THREADS, lds, s>>>(x, ld, r, temp, temp0, noise, V, slices, slice, parts, \
                                                                     choice, step)
  if (mode == CH_CDF) {
    VK_SLICES(false, false);
    choose_cdf_kernel<T><<<static_cast<unsigned>(B), CH_THREADS, lds, s>>>(x, ld, r, temp, temp0, noise, V, slices, slice,
                                                                       parts, choice, step);
  } else if (slices == 1) {
    if (mode == CH_GUMBEL)
      VK_SLICES(true, true);
    else
      VK_SLICES(false, true);
  } else if (mode == CH_GUMBEL) {
    VK_SLICES(true, false);
    choose_join_kernel<true><<<join, 256, 0, s>>>(parts, temp, temp0, B, V, slices, choice, step);
  } else {
    VK_SLICES(false, false);
    choose_join_kernel<false><<<join, 256, 0, s>>>(parts, temp, temp0, B, V, slices, choice, step);
  }
#undef VK_SLICES
  return launch_status("choose_tokens");
}

}  // namespace vk

using namespace vk;

extern "C" int vk_process_logits(const void *logits, int32_t dtype, int64_t ld, const int64_t *hist, int64_t hist_ld,
                                 int64_t hist_cols, const int32_t *hist_len, const float *rep, float rep0,
                                 const float *pres, float pres0, const float *freq, float freq0, const float *bias,
                                 int64_t bias_ld, const uint32_t *allowed, int64_t allowed_ld, int64_t n_allowed,
                                 const int32_t *allowed_rows, void *out, int32_t out_dtype, int64_t out_ld, int64_t B,
                                 int32_t V, void *stream) {
  int rc = check_logits(logits, dtype, ld, B, V, "process_logits");
  if (rc != VK_OK) return rc;
  VK_CHECK_ARG(out_dtype == VK_DTYPE_BF16 || out_dtype == VK_DTYPE_F32, "process_logits: out bf16 or fp32");
  VK_CHECK_ARG((B == 0 || out != nullptr) && out_ld >= V, "process_logits: out");
  VK_CHECK_ARG(out != logits || B == 0 || (out_dtype == dtype && out_ld == ld),
               "process_logits: in place needs one dtype and row stride");
  const Rules r = {hist, hist_ld, hist_cols, hist_len, nullptr, nullptr, rep, pres, freq, rep0, pres0, freq0, bias,
                   bias_ld, allowed, allowed_ld, n_allowed, allowed_rows, nullptr, nullptr};
  rc = check_rules(r, B, V, "process_logits");
  if (rc != VK_OK || B == 0) return rc;
  int slices, slice;
  slice_plan(B, V, &slices, &slice);
  const size_t lds = hist ? static_cast<size_t>(slice) * 2 : 0;
  const unsigned grid = static_cast<unsigned>(B * slices);
  hipStream_t s = VK_STREAM(stream);
  const bool lf = dtype == VK_DTYPE_F32, of = out_dtype == VK_DTYPE_F32;
#define VK_PROCESS(T, OT)                                                                                              \
  process_logits_kernel<T, OT><<<grid, CH_THREADS, lds, s>>>(static_cast<const T *>(logits), ld, r, V, slices, slice,  \
                                                             static_cast<OT *>(out), out_ld)
  if (lf && of)
    VK_PROCESS(float, float);
  else if (lf)
    VK_PROCESS(float, bf16_t);
  else if (of)
    VK_PROCESS(bf16_t, float);
  else
    VK_PROCESS(bf16_t, bf16_t);
#undef VK_PROCESS
  return launch_status("process_logits");
}

extern "C" int vk_choose_tokens_workspace(int64_t B, int32_t V, int64_t *bytes) {
  VK_CHECK_ARG(bytes && B >= 0 && V > 0, "choose_tokens_workspace: bad arguments");
  int slices = 0, slice = 0;
  if (B > 0) slice_plan(B, V, &slices, &slice);
  *bytes = B * slices * static_cast<int64_t>(sizeof(Part));
  return VK_OK;
}

static int choose(const void *logits, int32_t dtype, int64_t ld, const Rules &r, const float *temp, float temp0,
                  int32_t mode, const Noise &noise, const Choice &choice, const Step &step, int64_t B, int32_t V,
                  void *workspace, int64_t workspace_bytes, void *stream, const char *what) {
  int rc = check_logits(logits, dtype, ld, B, V, what);
  if (rc != VK_OK) return rc;
  rc = check_rules(r, B, V, what);
  if (rc != VK_OK) return rc;
  VK_CHECK_ARG(mode == CH_GREEDY || mode == CH_GUMBEL || mode == CH_CDF, "%s: mode 0 (greedy), 1 (Gumbel) or 2 (inverse CDF)",
               what);
  const int64_t per = mode == CH_GUMBEL ? V : 1;
  VK_CHECK_ARG(mode == CH_GREEDY || (noise.u != nullptr && noise.cols > 0 && noise.ld >= noise.cols * per),
               "%s: sampling needs uniforms, rows of columns x %lld", what, static_cast<long long>(per));
  if (B == 0) return VK_OK;
  int64_t need = 0;
  rc = vk_choose_tokens_workspace(B, V, &need);
  if (rc != VK_OK) return rc;
  VK_CHECK_ARG(workspace && vk_aligned16(workspace) && workspace_bytes >= need,
               "%s: a 16-byte aligned workspace of %lld bytes needed", what, static_cast<long long>(need));
  Part *parts = static_cast<Part *>(workspace);
  return dtype == VK_DTYPE_F32 ? launch_choose<float>(logits, ld, r, temp, temp0, mode, noise, B, V, parts, choice, step,
                                                      VK_STREAM(stream))
                               : launch_choose<bf16_t>(logits, ld, r, temp, temp0, mode, noise, B, V, parts, choice, step,
                                                       VK_STREAM(stream));
}

extern "C" int vk_choose_tokens(const void *logits, int32_t dtype, int64_t ld, const int64_t *hist, int64_t hist_ld,
                                int64_t hist_cols, const int32_t *hist_len, const float *rep, float rep0,
                                const float *pres, float pres0, const float *freq, float freq0, const float *bias,
                                int64_t bias_ld, const uint32_t *allowed, int64_t allowed_ld, int64_t n_allowed,
                                const int32_t *allowed_rows, const float *temp, float temp0, int32_t mode,
                                const float *uniforms, int64_t u_ld, int64_t fallback, int64_t *token, float *logp,
                                int64_t B, int32_t V, void *workspace, int64_t workspace_bytes, void *stream) {
  VK_CHECK_ARG(B <= 0 || token != nullptr, "choose_tokens: null pointer");
  const Rules r = {hist, hist_ld, hist_cols, hist_len, nullptr, nullptr, rep, pres, freq, rep0, pres0, freq0, bias,
                   bias_ld, allowed, allowed_ld, n_allowed, allowed_rows, nullptr, nullptr};
  return choose(logits, dtype, ld, r, temp, temp0, mode, Noise{uniforms, u_ld, 1}, Choice{token, logp, 0, fallback}, Step{},
                B, V, workspace, workspace_bytes, stream, "choose_tokens");
}

extern "C" int vk_choose_update(const void *logits, int32_t dtype, int64_t ld, float rep0, float pres0, float freq0,
                                const float *bias, const uint32_t *allowed, int64_t allowed_ld, int64_t n_allowed,
                                const int32_t *token_rows, const uint8_t *is_tail, const uint8_t *is_homo,
                                int32_t homo_stop, float temperature, int32_t mode, const float *uniforms, int64_t u_ld,
                                int64_t u_cols, int64_t *tok, int64_t *run, int64_t *pos, const int64_t *plen,
                                const int64_t *rope_off, const int64_t *cache_base, int64_t *out, int64_t out_stride,
                                int64_t out_cols, int32_t *pos32, int32_t *seqlens, int32_t *rpos32, float *logp,
                                int64_t logp_stride, int64_t B, int32_t V, int32_t eos, int32_t pad, void *workspace,
                                int64_t workspace_bytes, void *stream) {
  VK_CHECK_ARG(bias && is_tail && is_homo && tok && pos && out, "choose_update: null pointer");
  VK_CHECK_ARG(homo_stop <= 0 || run != nullptr, "choose_update: homopolymer rule needs run");
  VK_CHECK_ARG(out_cols > 0 && out_stride >= out_cols, "choose_update: output rows");
  VK_CHECK_ARG(logp_stride == 0 || logp_stride >= out_cols, "choose_update: logp_stride must be 0 or >= out_cols");
  VK_CHECK_ARG(allowed == nullptr || token_rows != nullptr, "choose_update: masks need the mask row of each token");
  VK_CHECK_ARG(rep0 > 0.f, "choose_update: the repetition penalty must be positive");
  // the tokens produced so far, out[b, 0 .. pos - plen - 1], are the history
  const bool penal = rep0 != 1.f || pres0 != 0.f || freq0 != 0.f;
  const Rules r = {penal ? out : nullptr, out_stride, out_cols, nullptr, pos, plen, nullptr, nullptr, nullptr, rep0, pres0,
                   freq0, bias, 0, allowed, allowed_ld, n_allowed, nullptr, token_rows, tok};
  const Step step = {{tok, run, pos, cache_base, out, out_stride, out_cols, pos32, seqlens, rpos32, homo_stop, eos, pad},
                     is_tail, is_homo, plen, rope_off};
  return choose(logits, dtype, ld, r, nullptr, temperature, mode, Noise{uniforms, u_ld, u_cols},
                Choice{nullptr, logp, logp_stride, pad}, step, B, V, workspace, workspace_bytes, stream, "choose_update");
}
