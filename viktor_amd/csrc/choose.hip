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

// cnt: 16-bit counts, two a word, of tokens v0 .. v0 + slice - 1 in hist[0 .. len - 1]. Ends with a barrier.
__device__ __forceinline__ void count_history(uint32_t *cnt, const int64_t *hist, int len, int v0, int slice) {
  for (int i = threadIdx.x; i < (slice + 1) / 2; i += CH_THREADS) cnt[i] = 0;
  __syncthreads();
  for (int t = threadIdx.x; t < len; t += CH_THREADS) {
    const int64_t rel = hist[t] - v0;
    if (rel >= 0 && rel < slice) atomicAdd(&cnt[rel >> 1], (rel & 1) ? 0x10000u : 1u);
  }
  __syncthreads();
}

// The rules on N tokens from v (N divides 8 and v: one mask word; `have` of them exist).
template <int N>
__device__ __forceinline__ void apply_rules(float (&z)[N], const RowRules &r, const uint32_t *cnt, int rel, int v,
                                            int have) {
#pragma clang fp contract(off)
  if (r.len > 0) {
    uint32_t w[N / 2], any = 0;
#pragma unroll
    for (int k = 0; k < N / 2; ++k) any |= w[k] = cnt[rel / 2 + k];
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
  if (r.bias != nullptr) {
    float bv[N];
    if (have == N) {
      load_row<N>(r.bias + v, bv);
    } else {
      for (int k = 0; k < N; ++k) bv[k] = k < have ? r.bias[v + k] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] = z[k] + bv[k];
  }
  if (r.allowed != nullptr) {
    const uint32_t bits = r.allowed[v >> 5] >> (v & 31);
#pragma unroll
    for (int k = 0; k < N; ++k) z[k] = (bits >> k) & 1 ? z[k] : -INFINITY;
  }
}

template <int N, typename T>
__device__ __forceinline__ int load_some(const T *row, int v, int V, float (&z)[N]) {
  const int have = V - v < N ? V - v : N;
  if (have == N) {
    load_row<N>(row + v, z);
  } else {
    for (int k = 0; k < N; ++k) z[k] = k < have ? load_one(row + v + k) : -INFINITY;
  }
  return have;
}

// grid: B x slices workgroups, a sequence's slices side by side. out may be logits.
template <typename T, typename OT>
__global__ __launch_bounds__(CH_THREADS) void process_logits_kernel(const T *logits, int64_t ld, Rules rules, int V,
                                                                    int slices, int slice, OT *out, int64_t out_ld) {
  extern __shared__ uint32_t cnt[];
  constexpr int N = 16 / sizeof(T);
  const int64_t b = blockIdx.x / slices;
  const int v0 = static_cast<int>(blockIdx.x % slices) * slice, v1 = V - v0 < slice ? V : v0 + slice;
  const RowRules r = row_rules(rules, b, V);
  if (r.len > 0) count_history(cnt, r.hist, r.len, v0, slice);
  const T *row = logits + b * ld;
  OT *dst = out + b * out_ld;
  for (int v = v0 + threadIdx.x * N; v < v1; v += CH_THREADS * N) {
    float z[N];
    const int have = load_some<N>(row, v, V, z);
    apply_rules<N>(z, r, cnt, v - v0, v, have);
    if (have == N) {
      store_row<N>(dst + v, z);
    } else {
      for (int k = 0; k < have; ++k) store_one(dst + v + k, z[k]);
    }
  }
}

// ---- the choice --------------------------------------------------------------------------------------------------------

enum { CH_GREEDY = 0, CH_GUMBEL = 1, CH_CDF = 2 };

struct Best {
  float s;    // its score in fp32 (Gumbel: within score_slack of the exact one)
  float z;    // its logit after the rules, before the temperature
  float u;    // its uniform
  int32_t v;  // -1: none yet
};

struct Part {
  float m, sum;  // max of z' (at least -FLT_MAX) and sum of exp(z' - m)
  Best best;
};

// How far the fp32 score of a token can be from the exact one: rounding of z' and of the sum (1.2e-7 of its size each),
// and of the two logarithms.
__device__ __forceinline__ float score_slack(float s) { return 1e-5f + 1e-6f * fabsf(s); }

// The exact score: z' rounded to fp32, the noise in 64 bits.
__device__ __forceinline__ double exact_score(const Best &a, float T) {
  return static_cast<double>(a.z / T) - log(-log(fmax(static_cast<double>(a.u), 1e-20)));
}

// Whether b comes before a. Gumbel scores that fp32 cannot order are compared in 64 bits.
template <bool GUMBEL>
__device__ __forceinline__ bool better(const Best &a, const Best &b, float T) {
  if (b.v < 0) return false;
  if (a.v < 0) return true;
  if (GUMBEL && T > 0.f) {
    const float d = b.s - a.s;
    if (fabsf(d) > 2.f * score_slack(fmaxf(fabsf(a.s), fabsf(b.s)))) return d > 0.f;
    const double ea = exact_score(a, T), eb = exact_score(b, T);
    return eb > ea || (eb == ea && b.v < a.v);
  }
  return b.s > a.s || (b.s == a.s && b.v < a.v);
}

__device__ __forceinline__ void join_sums(float &m, float &sum, float m2, float sum2) {
  const float M = fmaxf(m, m2);
  sum = sum * __expf(m - M) + sum2 * __expf(m2 - M);
  m = M;
}

template <bool GUMBEL>
__device__ __forceinline__ void join_lanes(Part &p, float T) {
#pragma unroll 1
  for (int o = 32; o > 0; o >>= 1) {
    Part q;
    q.m = __shfl_xor(p.m, o, 64);
    q.sum = __shfl_xor(p.sum, o, 64);
    q.best.s = __shfl_xor(p.best.s, o, 64);
    q.best.z = __shfl_xor(p.best.z, o, 64);
    q.best.u = __shfl_xor(p.best.u, o, 64);
    q.best.v = __shfl_xor(p.best.v, o, 64);
    join_sums(p.m, p.sum, q.m, q.sum);
    if (better<GUMBEL>(p.best, q.best, T)) p.best = q.best;
  }
}

// A NaN becomes -inf, +inf the largest finite value.
__device__ __forceinline__ float tame(float z) { return fminf(fmaxf(z, -INFINITY), FLT_MAX); }

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

template <typename T, bool GUMBEL>
__global__ __launch_bounds__(CH_THREADS) void choose_slices_kernel(const T *__restrict__ logits, int64_t ld, Rules rules,
                                                                   const float *__restrict__ temp, float temp0,
                                                                   Noise noise, int V, int slices, int slice, Part *__restrict__ parts) {
  extern __shared__ uint32_t cnt[];
  __shared__ Part red[CH_THREADS / 64];
  constexpr int N = 16 / sizeof(T);
  const int64_t b = blockIdx.x / slices;
  const int v0 = static_cast<int>(blockIdx.x % slices) * slice, v1 = V - v0 < slice ? V : v0 + slice;
  const RowRules r = row_rules(rules, b, V);
  const float temperature = temp ? temp[b] : temp0;
  const float inv = temperature > 0.f ? 1.f / temperature : 1.f;
  const bool noisy = GUMBEL && temperature > 0.f;
  if (r.len > 0) count_history(cnt, r.hist, r.len, v0, slice);
  const T *row = logits + b * ld;
  const float *urow = noisy ? noise_at(noise, rules, b, V) : nullptr;
  Part p = {-FLT_MAX, 0.f, {-INFINITY, 0.f, 0.f, -1}};
  for (int v = v0 + threadIdx.x * N; v < v1; v += CH_THREADS * N) {
    float z[N], u[N];
    const int have = load_some<N>(row, v, V, z);
    if (noisy) load_some<N>(urow, v, V, u);
    apply_rules<N>(z, r, cnt, v - v0, v, have);
    float q[N], m = p.m;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      z[k] = tame(z[k]);
      q[k] = tame(z[k] * inv);
      m = fmaxf(m, q[k]);
    }
    p.sum *= __expf(p.m - m);
    p.m = m;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      p.sum += __expf(q[k] - m);
      if (z[k] == -INFINITY) continue;
      const Best c = {noisy ? q[k] - logf(-logf(fmaxf(u[k], 1e-20f))) : q[k], z[k], noisy ? u[k] : 0.f, v + k};
      if (better<GUMBEL>(p.best, c, temperature)) p.best = c;
    }
  }
  join_lanes<GUMBEL>(p, temperature);
  const int lane = threadIdx.x & 63;
  if (lane == 0) red[threadIdx.x >> 6] = p;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < CH_THREADS / 64; ++w) {
      join_sums(p.m, p.sum, red[w].m, red[w].sum);
      if (better<GUMBEL>(p.best, red[w].best, temperature)) p.best = red[w].best;
    }
    parts[blockIdx.x] = p;
  }
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

// One wavefront per sequence joins its slices in slice order.
template <bool GUMBEL>
__global__ __launch_bounds__(256) void choose_join_kernel(const Part *__restrict__ parts, const float *__restrict__ temp,
                                                          float temp0, int64_t B, int V, int slices, Choice choice,
                                                          Step step) {
  const int64_t b = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (b >= B) return;
  const int lane = threadIdx.x & 63;
  const float temperature = temp ? temp[b] : temp0;
  Part p = {-FLT_MAX, 0.f, {-INFINITY, 0.f, 0.f, -1}};
  for (int s = lane; s < slices; s += 64) {
    const Part q = parts[b * slices + s];
    join_sums(p.m, p.sum, q.m, q.sum);
    if (better<GUMBEL>(p.best, q.best, temperature)) p.best = q.best;
  }
  join_lanes<GUMBEL>(p, temperature);
  if (lane != 0) return;
  const float zt = temperature > 0.f ? tame(p.best.z / temperature) : p.best.z;
  finish_row(choice, step, b, V, p.best.v, (zt - p.m) - logf(p.sum));
}

// Inverse CDF: one workgroup per sequence finds the slice that u falls into from the slices' sums (64 bits), then walks
// that slice in token order, CH_THREADS x N tokens a round. A row with temperature <= 0 takes the greedy choice.
template <typename T>
__global__ __launch_bounds__(CH_THREADS) void choose_cdf_kernel(const T *__restrict__ logits, int64_t ld, Rules rules,
                                                                const float *__restrict__ temp, float temp0,
                                                                Noise noise, int V, int slices, int slice,
                                                                const Part *__restrict__ parts,
                                                                Choice choice, Step step) {
  extern __shared__ uint32_t cnt[];
  __shared__ double wave_total[CH_THREADS / 64];
  __shared__ int found, last;
  constexpr int N = 16 / sizeof(T);
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const float temperature = temp ? temp[b] : temp0;
  const float inv = temperature > 0.f ? 1.f / temperature : 1.f;
  const Part *mine = parts + b * slices;
  // every thread joins the slices the same way
  float M = -FLT_MAX;
  Best best = {-INFINITY, 0.f, 0.f, -1};
  for (int s = 0; s < slices; ++s) {
    M = fmaxf(M, mine[s].m);
    if (better<false>(best, mine[s].best, 0.f)) best = mine[s].best;
  }
  double total = 0.;
  for (int s = 0; s < slices; ++s) total += static_cast<double>(mine[s].sum * __expf(mine[s].m - M));
  int pick = best.v;
  if (best.v >= 0 && temperature > 0.f) {
    const double target = static_cast<double>(*noise_at(noise, rules, b, 1)) * total;
    double before = 0.;
    int at = -1, filled = 0;
    double base = 0.;
    for (int s = 0; s < slices; ++s) {
      const double w = static_cast<double>(mine[s].sum * __expf(mine[s].m - M));
      if (at < 0 && w > 0.) {
        filled = s;
        base = before;
        if (target < before + w) at = s;
      }
      before += w;
    }
    if (at < 0) at = filled;  // rounding, or a uniform of 1: the last slice with any weight
    const RowRules r = row_rules(rules, b, V);
    const int v0 = at * slice, v1 = V - v0 < slice ? V : v0 + slice;
    if (tid == 0) {
      found = 0x7fffffff;
      last = -1;
    }
    __syncthreads();
    if (r.len > 0) count_history(cnt, r.hist, r.len, v0, slice);
    const T *row = logits + b * ld;
    double run = base;
    for (int w0 = v0; w0 < v1; w0 += CH_THREADS * N) {
      const int v = w0 + tid * N;
      double e[N], sum = 0.;
      int top = -1;
#pragma unroll
      for (int k = 0; k < N; ++k) e[k] = 0.;
      if (v < v1) {
        float z[N];
        const int have = load_some<N>(row, v, V, z);
        apply_rules<N>(z, r, cnt, v - v0, v, have);
#pragma unroll
        for (int k = 0; k < N; ++k) {
          e[k] = static_cast<double>(__expf(tame(tame(z[k]) * inv) - M));
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
      double left = run;
      for (int w = 0; w < CH_THREADS / 64; ++w) {
        if (w < wid) left += wave_total[w];
        run += wave_total[w];
      }
      left += inc - sum;
      double cdf = left;
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
    pick = found != 0x7fffffff ? found : last;
  }
  if (tid != 0) return;
  float logp = -INFINITY;
  if (pick >= 0) {  // the choice's own logit again
    const RowRules r = row_rules(rules, b, V);
    const int v = pick & ~(N - 1);
    float z[N];
    const int have = load_some<N>(logits + b * ld, v, V, z);
    if (best.v >= 0 && temperature > 0.f) {
      apply_rules<N>(z, r, cnt, v % slice, v, have);  // (slices start at multiples of the slice)
      logp = (tame(tame(z[pick - v]) / temperature) - M) - logf(static_cast<float>(total));
    } else {
      logp = (best.z - M) - logf(static_cast<float>(total));
    }
  }
  finish_row(choice, step, b, V, pick, logp);
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
  if (mode == CH_GUMBEL) {
    choose_slices_kernel<T, true><<<grid, CH_THREADS, lds, s>>>(x, ld, r, temp, temp0, noise, V, slices, slice, parts);
    choose_join_kernel<true><<<join, 256, 0, s>>>(parts, temp, temp0, B, V, slices, choice, step);
  } else {
    choose_slices_kernel<T, false><<<grid, CH_THREADS, lds, s>>>(x, ld, r, temp, temp0, noise, V, slices, slice, parts);
    if (mode == CH_CDF)
      choose_cdf_kernel<T><<<static_cast<unsigned>(B), CH_THREADS, lds, s>>>(x, ld, r, temp, temp0, noise, V, slices, slice,
                                                                         parts, choice, step);
    else
      choose_join_kernel<false><<<join, 256, 0, s>>>(parts, temp, temp0, B, V, slices, choice, step);
  }
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
