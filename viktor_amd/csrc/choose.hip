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
// A workgroup takes one slice of one sequence's vocabulary. The history's tokens of the slice are gathered in LDS (Seen),
// so no count per (sequence, token) exists in memory and the streaming pass over the logits knows of the history only that
// a token is left out: a distinct token of it is computed once, by one thread. Logits are loaded a batch ahead of their use.
// The choice gives (max, sum of exponentials at it, best) per slice, joined by one wavefront per sequence, or takes a whole
// row per workgroup of 512 threads and finishes it (make_plan).
//
// What bounds them: one sequence, the launch and the chain of loads (process 4.8 us at 5463 tokens, choice 8.9 us at 87383
// in two launches; in a graph); a batch, memory, and before it the gathering and the bias, which is read from the L2s as
// often as there are sequences (of 179 MB of fp32 logits and as many of bias, 192 MB pass the L2s in all). 512 x 87383
// logits, us (a plain read of the fp32 ones takes 26.5, a copy of the bf16 ones 31 to 36):
//                 no rules   bias   mask   history of 256   all
//   process bf16      37      45     38         43           51 (46.4 from logits that are not in a cache)
//   process fp32      74      79     77         81           84
//   greedy fp32       31.5    37     33         35           42
//   greedy bf16       23.7    33     27         27           37
// Histories of 1, 64, 1024, 2048, 4096 columns take processed bf16 logits 47, 50, 56, 68, 86: each slice of a row reads all
// of its sequence's history.
// The inverse CDF keeps its sums by batch or slice and reads only the batch or slice that the uniform falls into again: with
// a bias 49 (fp32) and 42 (bf16), with all rules 56 and 47; 5463 tokens 23 against 10 greedy, since a row of one batch is
// loaded, ruled and scanned a second time.
// A decode step (choose_update), us, greedy / Gumbel / inverse CDF with a bias, then with penalties and a grammar too, fp32:
// 1 x 5463 5.2 / 7.1 / 13.8, 7.1 / 9.3 / 16.6; 64 x 5463 5.9 / 7.8 / 14.5, 8.0 / 10.2 / 17.7; 512 x 5463 8.0 / 11.3 / 19.6,
// 10.8 / 14.7 / 23.3; 64 x 87383 13.1 / 18.8 / 27.0, 16.1 / 21.7 / 33.3; 512 x 87383 39.2 / 63.6 / 51.6, 43.3 / 71.0 / 58.4.
// Measured and not taken: bias and mask loaded a batch ahead (process fp32 -4, all bf16 +2), two sequences a workgroup that
// share the bias (bf16 -0.6, fp32 +5), 8-byte loads of bf16 (+1 to +2), 1024 threads a row (+5), two batches ahead (+1 to
// +2).
#include <float.h>
#include <math.h>

#include <type_traits>

#include "decode_state.h"
#include "row_access.h"

namespace vk {

constexpr int CH_THREADS = 256;
constexpr int CH_THREADS_ONE = 512;  // of a workgroup that takes a whole row
constexpr int CH_WHOLE = 1 << 17;    // tokens of such a row at most, where it has more than one slice: 16 KB of LDS bits
// Tokens of a row that one workgroup takes at any batch: it spares the join's launch, and the inverse CDF the history's
// second gathering. All rules, fp32, us in a graph, 1 / 8 / 77 sequences, whole against slices:
//             greedy                              Gumbel                               inverse CDF
//    9001  7.5  7.8  8.8 : 8.6 9.3 10.1   10.2 10.5 11.8 : 10.3 11.2 12.2   14.4 18.5 20.2 : 17.3 21.7 22.9
//   21847  8.4  9.5 10.8 : 8.6 9.4 10.9   12.5 13.3 14.8 : 10.4 11.7 14.2   15.6 19.9 22.1 : 17.2 21.2 23.4
//   32000  9.9 11.0 12.1 : 8.5 9.5 12.5   14.9 15.9 17.2 : 10.4 11.6 17.1   17.1 21.5 23.4 : 16.7 21.3 31.6
//   43000 11.4 13.7 14.9 : 8.6 9.4 12.8   18.0 21.2 22.6 : 10.4 11.7 17.6   19.2 24.8 26.6 : 17.2 21.2 31.4
// One border for all three: the Gumbel choice of a few sequences gains 2 us from slices at 21847 already (it computes more
// a token), the inverse CDF of 77 loses 5 by them at 43000.
constexpr int CH_SMALL = 32768;
constexpr int CH_SLICE = 8192;       // tokens of a slice at most (512 x 87383 bf16, processed: 51 us; of 4096 55, 16384 57)
// History columns at most whose counts are hashed, 32 KB of LDS at the most. 512 x 87383 bf16, processed, histories of 256:
// 51 us, counted by token 57 (32 KB to clear and to hold); of 2048: 68 and 66.
constexpr int CH_HASH_MAX = 2048;
constexpr int CH_HIST_MAX = 65535;
constexpr int32_t CH_V_MAX = 1 << 30;

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

// How a call is cut: slices of `slice` tokens per sequence, and the history's table (Seen).
struct Plan {
  int slices, slice, slots, listed;
  bool hashed, one;
};

struct RowRules {
  const int64_t *hist;
  int len;  // 0: no penalties
  float rep, pres, freq;
  const float *bias;
  const uint32_t *allowed;
};

// What a pointer that is not given is read from instead, so that a row's scalars are loaded side by side.
__device__ const int64_t kNothing[1] = {0};

template <typename P>
__device__ __forceinline__ P at_or_zero(const P *p, int64_t i) {
  return *(p != nullptr ? p + i : reinterpret_cast<const P *>(kNothing));
}

__device__ __forceinline__ RowRules row_rules(const Rules &r, int64_t b, int V) {
  const float rep = at_or_zero(r.rep, b), pres = at_or_zero(r.pres, b), freq = at_or_zero(r.freq, b);
  const int32_t len = at_or_zero(r.len, b), arow = at_or_zero(r.arow, b);
  const int64_t pos = at_or_zero(r.pos, b), plen = at_or_zero(r.plen, b), tok = at_or_zero(r.tok, b);
  RowRules o = {};
  if (r.hist != nullptr) {
    o.rep = r.rep ? rep : r.rep0;
    o.pres = r.pres ? pres : r.pres0;
    o.freq = r.freq ? freq : r.freq0;
    int64_t n = r.len ? len : pos - plen;
    n = n < 0 ? 0 : (n > r.hist_cols ? r.hist_cols : n);
    o.hist = r.hist + b * r.hist_ld;
    // repetition 1 divides and multiplies by one, and the others subtract zero: nothing to count
    o.len = o.rep == 1.f && o.pres == 0.f && o.freq == 0.f ? 0 : static_cast<int>(n);
  }
  o.bias = r.bias ? r.bias + b * r.bias_ld : nullptr;
  if (r.allowed != nullptr) {
    int64_t a = b;
    if (r.token_row != nullptr)
      a = tok >= 0 && tok < V ? r.token_row[tok] : -1;
    else if (r.arow != nullptr)
      a = arow;
    else if (r.n_allowed == 1)
      a = 0;
    if (a >= 0 && a < r.n_allowed) o.allowed = r.allowed + a * r.allowed_ld;
  }
  return o;
}

// The history's tokens of a slice, in dynamic LDS: a bit per token of the slice, and how often each occurs, in a hash
// table of `slots` (a power of two, at least twice the history's columns) or, for long histories, by token (slots = slice).
// Every distinct token is then one slot, on a list (of at most `listed`, in any order), whose logit one thread computes;
// the streaming pass leaves tokens with a bit out. Without the list the threads went through all slots, a wait for a
// logit at nearly every step: 119 us for 512 x 87383 bf16 logits with histories of 2048, and 55 with 256.
template <int THREADS>
struct Seen {
  uint32_t *bits, *count, *key, *distinct;  // key: null by token
  uint16_t *list;
  int slots, shift;
  static constexpr uint32_t kEmpty = 0xffffffffu;

  __device__ __forceinline__ Seen(uint32_t *lds, const Plan &p)
      : bits(lds), count(lds + p.slice / 32), key(p.hashed ? count + p.slots : nullptr),
        distinct(count + (p.hashed ? 2 : 1) * p.slots), list(reinterpret_cast<uint16_t *>(distinct + 4)), slots(p.slots),
        shift(__clz(p.slots) + 1) {}
  __device__ __forceinline__ bool has(int rel) const { return (bits[rel >> 5] >> (rel & 31)) & 1; }
  // The slot of a token of the slice; of one that is not there, a new one (at most half of them get used).
  __device__ __forceinline__ int slot(uint32_t rel) const {
    if (key == nullptr) return static_cast<int>(rel);
    uint32_t h = (rel * 0x9E3779B1u) >> shift;
    while (true) {
      const uint32_t old = atomicCAS(&key[h], kEmpty, rel);
      if (old == kEmpty || old == rel) return static_cast<int>(h);
      h = (h + 1) & (slots - 1);
    }
  }
  // Of tokens v0 .. v1 - 1. Ends with a barrier.
  __device__ __forceinline__ void fill(const int64_t *hist, int len, int v0, int v1, int slice) const {
    constexpr int U = 4;  // of a thread's tokens in flight, the first ones while the table is cleared
    const int tid = threadIdx.x;
    int64_t h[U];
    auto load = [&](int t0) {
#pragma unroll
      for (int u = 0; u < U; ++u) h[u] = hist[min(t0 + u * THREADS, len - 1)];
    };
    load(tid);
    if (tid == 0) *distinct = 0;
    for (int i = tid; i < (slice / 32 + slots) / 4; i += THREADS) reinterpret_cast<u32x4 *>(bits)[i] = u32x4{0u, 0u, 0u, 0u};
    if (key != nullptr)
      for (int i = tid; i < slots / 4; i += THREADS)
        reinterpret_cast<u32x4 *>(key)[i] = u32x4{kEmpty, kEmpty, kEmpty, kEmpty};
    __syncthreads();
    for (int t0 = tid; t0 < len; t0 += U * THREADS) {
      if (t0 != tid) load(t0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint64_t far = static_cast<uint64_t>(h[u]) - static_cast<uint64_t>(v0);
        if (t0 + u * THREADS < len && far < static_cast<uint64_t>(v1 - v0)) {
          const uint32_t rel = static_cast<uint32_t>(far), bit = 1u << (rel & 31);
          const int at = slot(rel);
          atomicAdd(&count[at], 1u);
          if ((atomicOr(&bits[rel >> 5], bit) & bit) == 0) list[atomicAdd(distinct, 1u)] = static_cast<uint16_t>(at);
        }
      }
    }
    __syncthreads();
  }
  // This thread's distinct tokens, as f(token of the slice, its count's place).
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (uint32_t i = threadIdx.x; i < *distinct; i += THREADS) {
      const int at = list[i];
      f(static_cast<int>(key != nullptr ? key[at] : at), count[at]);
    }
  }
};

// One token's logit after the rules; count: its occurrences in the history.
template <typename T>
__device__ __forceinline__ float one_logit(const T *row, const RowRules &r, int v, uint32_t count) {
#pragma clang fp contract(off)
  float z = load_one(row + v);
  const float bias = r.bias != nullptr ? r.bias[v] : 0.f;
  const bool allowed = r.allowed == nullptr || ((r.allowed[v >> 5] >> (v & 31)) & 1);
  if (count > 0) {
    z = z > 0.f ? z / r.rep : z * r.rep;
    z = z - r.freq * static_cast<float>(count);
    z = z - r.pres;
  }
  if (r.bias != nullptr) z = z + bias;
  return allowed ? z : -INFINITY;
}

// What a thread takes of a workgroup's next 16 THREADS tokens: R vectors of N tokens, vector q at token
// first + q * THREADS * N + threadIdx.x * N. CUT: the row ends inside the batch; one that is cut (N does not divide V) is
// read token by token.
template <typename T, int THREADS>
struct Batch {
  static constexpr int N = 16 / sizeof(T), R = sizeof(T), STEP = THREADS * N, TOKENS = R * STEP;
  u32x4 raw[R];

  static __device__ __forceinline__ int token(int first, int q) {
    return first + q * STEP + static_cast<int>(threadIdx.x) * N;
  }
  // Where vector q is loaded from (V >= N): past the row's end, its last whole vector. So all loads are unconditional and
  // in bounds, and a wait for older loads can leave them in flight.
  static __device__ __forceinline__ int from(int first, int q, int V) { return min(token(first, q), V - N); }

  // (V >= N)
  __device__ __forceinline__ void load(const T *row, int first, int V) {
#pragma unroll
    for (int q = 0; q < R; ++q) raw[q] = stream_16(row + from(first, q, V));
  }

  // z: the batch's logits after bias and mask (-inf past the row's end). MORE: the next batch's logits are loaded as soon
  // as these are taken, behind this one's bias and mask. left_out: a bit per token of the slice from v0, of those that get
  // -inf too (null: none). All of a token's reasons for -inf are one bit, spread to a word and merged in: 2 instructions a
  // token.
  template <bool CUT, bool MORE>
  __device__ __forceinline__ void rules(float (&z)[R][N], const T *row, const RowRules &r, int first, int V,
                                        const uint32_t *left_out, int v0) {
#pragma clang fp contract(off)
#pragma unroll
    for (int q = 0; q < R; ++q)
#pragma unroll
      for (int k = 0; k < N; ++k)
        if constexpr (sizeof(T) == 4)
          z[q][k] = __uint_as_float(raw[q][k]);
        else
          z[q][k] = (k & 1) ? hi_bf(raw[q][k / 2]) : lo_bf(raw[q][k / 2]);
    float bias[R][N];
    uint32_t mask[R];
    if (r.bias != nullptr && !(CUT && V < N))
#pragma unroll
      for (int q = 0; q < R; ++q) load_row<N>(r.bias + (CUT ? from(first, q, V) : token(first, q)), bias[q]);
    if (r.allowed != nullptr)
#pragma unroll
      for (int q = 0; q < R; ++q) mask[q] = r.allowed[(CUT ? min(token(first, q), V - 1) : token(first, q)) >> 5];
    if (MORE) load(row, first + TOKENS, V);
    if (CUT) {
#pragma unroll
      for (int q = 0; q < R; ++q) {
        const int v = token(first, q);
        if (v < V && v > V - N)
          for (int k = 0; k < N; ++k) {
            const int at = v + k < V ? v + k : V - 1;
            z[q][k] = load_one(row + at);
            if (r.bias != nullptr) bias[q][k] = r.bias[at];
          }
      }
    }
    if (r.bias != nullptr)
#pragma unroll
      for (int q = 0; q < R; ++q)
#pragma unroll
        for (int k = 0; k < N; ++k) z[q][k] = z[q][k] + bias[q][k];
    const int lane_bit = (threadIdx.x * N) & 31;  // (first and STEP are multiples of 32)
    if (!CUT && r.allowed == nullptr && left_out == nullptr) return;
#pragma unroll
    for (int q = 0; q < R; ++q) {
      uint32_t keep = r.allowed != nullptr ? mask[q] >> lane_bit : ~0u;
      if (left_out != nullptr) keep &= ~(left_out[(token(first, q) - v0) >> 5] >> lane_bit);
      if (CUT) keep &= (1u << max(0, min(N, V - token(first, q)))) - 1;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const uint32_t whole = static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(keep), k, 1));
        z[q][k] = __uint_as_float((__float_as_uint(z[q][k]) & whole) | (0xff800000u & ~whole));
      }
    }
  }
};

template <typename T, typename OT, bool CUT, bool MORE>
__device__ __forceinline__ void process_batch(Batch<T, CH_THREADS> &x, const T *row, OT *dst, const RowRules &r, int w,
                                              int V) {
  using X = Batch<T, CH_THREADS>;
  float z[X::R][X::N];
  x.template rules<CUT, MORE>(z, row, r, w, V, nullptr, 0);
#pragma unroll
  for (int q = 0; q < X::R; ++q) {
    const int v = X::token(w, q);
    if (!CUT || v <= V - X::N)
      store_row<X::N>(dst + v, z[q]);
    else
      for (int k = 0; k < X::N && v + k < V; ++k) store_one(dst + v + k, z[q][k]);
  }
}

// grid: B x slices workgroups, a sequence's slices side by side. The logits of the history's tokens are computed from what
// was there before any store (out may be logits), and stored over what the streaming pass, which knows of no history, has
// put there.
template <typename T, typename OT>
__global__ __launch_bounds__(CH_THREADS) void process_logits_kernel(const T *logits, int64_t ld, Rules rules, int V,
                                                                    Plan plan, OT *out, int64_t out_ld) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  using X = Batch<T, CH_THREADS>;
  const int64_t b = blockIdx.x / plan.slices;
  const int v0 = static_cast<int>(blockIdx.x % plan.slices) * plan.slice, v1 = V - v0 < plan.slice ? V : v0 + plan.slice;
  const Seen<CH_THREADS> seen(lds, plan);
  const T *row = logits + b * ld;
  OT *dst = out + b * out_ld;
  X x;
  if (V >= X::N) x.load(row, v0, V);
  const RowRules r = row_rules(rules, b, V);
  if (r.len > 0) {
    seen.fill(r.hist, r.len, v0, v1, plan.slice);
    seen.each([&](int rel, uint32_t &count) { count = __float_as_uint(one_logit(row, r, v0 + rel, count)); });
    __syncthreads();
  }
  int w = v0;
  for (; w + X::TOKENS < v1; w += X::TOKENS) process_batch<T, OT, false, true>(x, row, dst, r, w, V);
  if (w + X::TOKENS <= V)
    process_batch<T, OT, false, false>(x, row, dst, r, w, V);
  else
    process_batch<T, OT, true, false>(x, row, dst, r, w, V);
  if (r.len > 0) {
    __syncthreads();
    seen.each([&](int rel, uint32_t z) { store_one(dst + v0 + rel, __uint_as_float(z)); });
  }
}

// ---- the choice --------------------------------------------------------------------------------------------------------

enum { CH_GREEDY = 0, CH_GUMBEL = 1, CH_CDF = 2 };

// A slice's result: the maximum of z (at least -FLT_MAX), the sum of exp((z - m) / T), and the best token v (-1: none).
// Its z is its logit after the rules; Gumbel: s its score in fp32 (within score_slack of the exact one), u its uniform.
struct Part {
  float m, sum, s, z, u;
  int32_t v;
};

// A thread's offer for the workgroup's best token.
struct Best {
  float s, z, u;
  int32_t v;
};

__device__ __forceinline__ Part no_part() { return {-FLT_MAX, 0.f, -INFINITY, -INFINITY, 0.f, -1}; }

// How far the fp32 score of a token can be from the exact one: the roundings of z' and of the sum (1.2e-7 of its size
// each), and of the two logarithms.
__device__ __forceinline__ float score_slack(float s) { return 1e-5f + 1e-6f * fabsf(s); }

// The least fp32 score that can be the best one where the largest fp32 score is `most` (a NaN for inf: any can).
__device__ __forceinline__ float contender_from(float most) { return most - 2.5f * score_slack(most); }

// The exact score: z' rounded to fp32 unless that overflows, the noise in 64 bits.
__device__ __forceinline__ double exact_score(float z, float u, float T) {
  const float q = z / T;
  const double scaled = fabsf(q) <= FLT_MAX ? static_cast<double>(q) : static_cast<double>(z) / T;
  return scaled - log(-log(fmax(static_cast<double>(u), 1e-20)));
}

struct Scale {
  float T, inv, L;  // the temperature, 1 / T (1 for a greedy row) and log2(e) / T, all kept finite
};

__device__ __forceinline__ Scale row_scale(const float *temp, float temp0, int64_t b) {
  Scale c;
  c.T = temp ? temp[b] : temp0;
  if (c.T > FLT_MAX) c.T = FLT_MAX;  // (an infinite one: -inf would become a NaN)
  c.inv = c.T > 0.f ? fminf(1.f / c.T, 0.5f * FLT_MAX) : 1.f;
  c.L = fminf(c.inv * 1.44269504f, 0.5f * FLT_MAX);
  return c;
}

// The score in fp32, from the hardware's base-2 logarithms. -inf for -inf.
__device__ __forceinline__ float gumbel_score(float z, float u, const Scale &c) {
  const float w = -0.693147181f * __builtin_amdgcn_logf(fmaxf(u, 1e-20f));
  return fmaf(z, c.inv, -0.693147181f * __builtin_amdgcn_logf(w));
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

__device__ __forceinline__ float wave_max_of(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = vmax2(v, __shfl_xor(v, o, 64));
  return v;
}

// What a thread knows of its tokens (without the history's): the maximum of z (at least -FLT_MAX), the sum of exponentials
// at it, the best logit or score with its first token, and the second best score. A batch that has nothing near the
// wavefront's best so far is not looked through for them (a thread's next best comes in most batches, a wavefront's in one
// of i at the i-th).
struct Mine {
  float m = -FLT_MAX, sum = 0.f, best = -INFINITY, second = -INFINITY, wave_best = -INFINITY;
  int v = -1;
};

// The uniforms of the batch to come (Gumbel; a greedy row's are loaded too, so that the loads are unconditional).
template <typename T, int THREADS, bool GUMBEL>
struct Uniforms {
  using X = Batch<T, THREADS>;
  float next[GUMBEL ? X::R : 1][X::N];
  __device__ __forceinline__ void load(const float *urow, int first, int V) {
    if constexpr (GUMBEL) {
#pragma unroll
      for (int q = 0; q < X::R; ++q) stream_row<X::N>(urow + X::from(first, q, V), next[q]);
    }
  }
  __device__ __forceinline__ void take(float (&u)[GUMBEL ? X::R : 1][X::N]) const {
    if constexpr (GUMBEL)
#pragma unroll
      for (int q = 0; q < X::R; ++q)
#pragma unroll
        for (int k = 0; k < X::N; ++k) u[q][k] = next[q][k];
  }
};

template <typename T, int THREADS, int MODE, bool CUT, bool MORE>
__device__ __forceinline__ void choose_batch(Batch<T, THREADS> &x, Uniforms<T, THREADS, MODE == CH_GUMBEL> &un,
                                             Mine &t, const T *row, const float *urow, const RowRules &r, const Scale &c,
                                             const Seen<THREADS> &s, int v0, int w, int V) {
  using X = Batch<T, THREADS>;
  constexpr bool GUMBEL = MODE == CH_GUMBEL;
  const bool noisy = GUMBEL && c.T > 0.f;
  float z[X::R][X::N], u[GUMBEL ? X::R : 1][X::N];
  un.take(u);
  x.template rules<CUT, MORE>(z, row, r, w, V, r.len > 0 ? s.bits : nullptr, v0);  // (the history's tokens: each())
  if (MORE) un.load(urow, w + X::TOKENS, V);
  float top = -INFINITY;
#pragma unroll
  for (int q = 0; q < X::R; ++q)
#pragma unroll
    for (int k = 0; k < X::N; k += 2) {
      z[q][k] = tame(z[q][k]);
      z[q][k + 1] = tame(z[q][k + 1]);
      top = vmax3(top, z[q][k], z[q][k + 1]);
    }
  if constexpr (MODE != CH_CDF) {
    const float m = vmax2(t.m, top);
    t.sum *= __builtin_amdgcn_exp2f((t.m - m) * c.L);
    t.m = m;
#pragma unroll
    for (int q = 0; q < X::R; ++q)
#pragma unroll
      for (int k = 0; k < X::N; ++k) t.sum += __builtin_amdgcn_exp2f((z[q][k] - m) * c.L);
  }
  if (noisy) {
    if constexpr (GUMBEL) {
      if (CUT)
#pragma unroll
        for (int q = 0; q < X::R; ++q) {
          const int v = X::token(w, q);
          if (v < V && v > V - X::N)
            for (int k = 0; k < X::N; ++k) u[q][k] = urow[v + k < V ? v + k : V - 1];
        }
      float most = -INFINITY;
#pragma unroll
      for (int q = 0; q < X::R; ++q)
#pragma unroll
        for (int k = 0; k < X::N; k += 2) {
          u[q][k] = gumbel_score(z[q][k], u[q][k], c);
          u[q][k + 1] = gumbel_score(z[q][k + 1], u[q][k + 1], c);
          most = vmax3(most, u[q][k], u[q][k + 1]);
        }
      if (__any(!(most < contender_from(t.wave_best)))) {
#pragma unroll
        for (int q = 0; q < X::R; ++q)
#pragma unroll
          for (int k = 0; k < X::N; ++k) {
            const float sc = u[q][k];
            t.second = fmaxf(t.second, fminf(t.best, sc));
            if (sc > t.best) {
              t.best = sc;
              t.v = X::token(w, q) + k;
            }
          }
        t.wave_best = wave_max_of(t.best);
      }
    }
  } else if (__any(top > t.wave_best)) {  // (a later batch's equal logit is behind the earlier one's)
    if (top > t.best) {
      t.v = 0x7fffffff;
      t.best = top;
#pragma unroll
      for (int q = X::R - 1; q >= 0; --q)
#pragma unroll
        for (int k = X::N - 1; k >= 0; --k) t.v = z[q][k] == top ? min(t.v, X::token(w, q) + k) : t.v;
    }
    t.wave_best = wave_max_of(t.best);
  }
  if constexpr (MODE == CH_CDF) {  // the wavefront's sum of the batch, at its largest logit so far
    t.m = vmax2(t.wave_best, -FLT_MAX);
    t.sum = 0.f;
#pragma unroll
    for (int q = 0; q < X::R; ++q)
#pragma unroll
      for (int k = 0; k < X::N; ++k) t.sum += __builtin_amdgcn_exp2f((z[q][k] - t.m) * c.L);
    t.sum = wave_sum(t.sum);
  }
}

// ---- the inverse CDF ---------------------------------------------------------------------------------------------------

// The history's logits of a slice, in place of their counts (between barriers).
template <typename T, int THREADS>
__device__ __forceinline__ void logits_for_counts(const Seen<THREADS> &s, const T *row, const RowRules &r, int v0) {
  s.each([&](int rel, uint32_t &count) { count = __float_as_uint(one_logit(row, r, v0 + rel, count)); });
}

// A weight exp((z - M) / T) of at most 1 in whole steps of 2^-40. The history's tokens are added up in these: which thread
// finds which of them first is not the same in every run, and the order of additions does not matter where they are exact
// (a slice's distinct tokens, at most 8192, come to 2^53 steps).
constexpr double STEPS = 1099511627776.;
__device__ __forceinline__ double weight_steps(float z, float M, const Scale &c) {
  return floor(static_cast<double>(__builtin_amdgcn_exp2f((z - M) * c.L)) * STEPS);
}

// What the workgroup's threads share while they look for the token that the target falls into.
template <int THREADS>
struct Walk {
  double segment[4 * (THREADS / 64)];  // sums of the wavefronts' tokens (R <= 4 times 64 N each), in token order
  int found, last;                     // the token; the last one with any weight so far
};

// A batch's weights exp((z - M) / T) in token order, after `run`: the first token whose running sum passes the target. Sums
// in 64 bits: a thread's N tokens, the wavefront's threads by a scan, and the wavefronts' segments one by one. Counts have
// been replaced by logits. Ends with a barrier.
template <typename T, int THREADS>
__device__ __forceinline__ void walk_batch(Batch<T, THREADS> &x, const T *row, const RowRules &r, const Scale &c,
                                           const Seen<THREADS> &s, int v0, int w, int V, float M, double target, double &run,
                                           Walk<THREADS> &shared) {
  using X = Batch<T, THREADS>;
  constexpr int WAVES = THREADS / 64;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  float z[X::R][X::N];
  double own[X::R], upto[X::R];
  x.template rules<true, false>(z, row, r, w, V, nullptr, 0);
#pragma unroll
  for (int q = 0; q < X::R; ++q) {
    if (r.len > 0) {
      const int rel = X::token(w, q) - v0;
      const uint32_t left = (s.bits[rel >> 5] >> (rel & 31)) & ((1u << X::N) - 1);
      if (left != 0)
#pragma unroll
        for (int k = 0; k < X::N; ++k)
          if ((left >> k) & 1) z[q][k] = __uint_as_float(s.count[s.slot(rel + k)]);
    }
    own[q] = 0.;
#pragma unroll
    for (int k = 0; k < X::N; ++k) {
      z[q][k] = __builtin_amdgcn_exp2f((tame(z[q][k]) - M) * c.L);
      own[q] += static_cast<double>(z[q][k]);
    }
    upto[q] = own[q];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(upto[q], o, 64);
      if (lane >= o) upto[q] += up;
    }
    if (lane == 63) shared.segment[q * WAVES + wid] = upto[q];
  }
  __syncthreads();
  int hit = 0x7fffffff, top = -1;
#pragma unroll
  for (int q = 0; q < X::R; ++q) {
    double cdf = run;
    for (int i = 0; i < WAVES; ++i) {
      if (i == wid) cdf = run;
      run += shared.segment[q * WAVES + i];
    }
    cdf += upto[q] - own[q];
#pragma unroll
    for (int k = 0; k < X::N; ++k) {
      cdf += static_cast<double>(z[q][k]);
      if (z[q][k] > 0.f) {
        top = X::token(w, q) + k;
        if (hit == 0x7fffffff && target < cdf) hit = top;
      }
    }
  }
  if (hit != 0x7fffffff) atomicMin(&shared.found, hit);
  if (top >= 0) atomicMax(&shared.last, top);
  __syncthreads();
}

// The end of it, by one thread: the token found, or the last with weight (rounding, or a uniform of 1).
template <typename T, int THREADS>
__device__ __forceinline__ void finish_walk(const Walk<THREADS> &shared, const T *row, const RowRules &r, const Scale &c,
                                            const Seen<THREADS> &s, int v0, int V, const Part &p, const Choice &choice,
                                            const Step &step, int64_t b) {
  const int pick = shared.found != 0x7fffffff ? shared.found : shared.last;
  if (pick < 0) {  // (what has weight holds a token with weight)
    finish_row(choice, step, b, V, p.v, logp_of(p.z, p, c));
  } else {
    const bool seen = r.len > 0 && s.has(pick - v0);
    const float z = seen ? __uint_as_float(s.count[s.slot(pick - v0)]) : one_logit(row, r, pick, 0);
    finish_row(choice, step, b, V, pick, logp_of(tame(z), p, c));
  }
}

// The whole row's sums by batch and wavefront, of a workgroup that takes a row.
template <int THREADS>
struct BatchSums {
  static constexpr int MOST = CH_WHOLE / (16 * THREADS);
  float sum[MOST][THREADS / 64], m[MOST][THREADS / 64];
  double total[MOST];    // of a batch at the row's maximum
  double history[MOST];  // of its history's tokens
  Walk<THREADS> walk;
};

// The choice from a row's sums by batch (p: its maximum and its first best token): the totals at the maximum, the batch that
// the target falls into, and the token in it.
template <typename T, int THREADS>
__device__ __forceinline__ void choose_from_sums(BatchSums<THREADS> &sums, Batch<T, THREADS> &x, const T *row,
                                                 const RowRules &r, const Scale &c, const Seen<THREADS> &s, int V,
                                                 int batches, Part p, const float *uniform, const Choice &choice,
                                                 const Step &step, int64_t b) {
  using X = Batch<T, THREADS>;
  constexpr int WAVES = THREADS / 64;
  const int tid = threadIdx.x;
  if (r.len > 0)
    s.each([&](int rel, uint32_t z) {
      atomicAdd(&sums.history[rel / X::TOKENS], weight_steps(__uint_as_float(z), p.m, c));
    });
  __syncthreads();
  if (tid < batches) {
    double total = sums.history[tid] / STEPS;
    for (int i = 0; i < WAVES; ++i)
      total += static_cast<double>(sums.sum[tid][i]) * __builtin_amdgcn_exp2f((sums.m[tid][i] - p.m) * c.L);
    sums.total[tid] = total;
  }
  __syncthreads();
  double total = 0.;
  for (int i = 0; i < batches; ++i) total += sums.total[i];
  p.sum = static_cast<float>(total);
  if (p.v < 0 || !(c.T > 0.f)) {
    if (tid == 0) finish_row(choice, step, b, V, p.v, logp_of(p.z, p, c));
    return;
  }
  // (rounding, or a uniform of 1: the last batch with any weight)
  const double target = static_cast<double>(*uniform) * total;
  int at = 0;
  double run = 0., before = 0.;
  for (int i = 0; i < batches; ++i)
    if (sums.total[i] > 0.) {
      at = i;
      run = before;
      before += sums.total[i];
      if (target < before) break;
    }
  if (V >= X::N) x.load(row, at * X::TOKENS, V);
  walk_batch(x, row, r, c, s, 0, at * X::TOKENS, V, p.m, target, run, sums.walk);
  if (tid == 0) finish_walk(sums.walk, row, r, c, s, 0, V, p, choice, step, b);
}

// One slice of one sequence, or with ONE the whole vocabulary and the step's end. The workgroup's best logit or score
// tells who can have the best token: the lowest token of the largest logit, or the threads within the scores' slack of
// the largest score. These read their token again and are compared exactly; one whose second score is as near goes
// through all of its tokens, its history's too, and so does every thread where all scores are below fp32's range. The sum is
// taken at the workgroup's maximum. Inverse CDF (ONE): the sums stay by batch, and the batch that the uniform falls into is
// walked.
template <typename T, int THREADS, int MODE, bool ONE>
__global__ __launch_bounds__(THREADS) void choose_slices_kernel(const T *__restrict__ logits, int64_t ld, Rules rules,
                                                                   const float *__restrict__ temp, float temp0,
                                                                   Noise noise, int V, Plan plan,
                                                                   Part *__restrict__ parts, Choice choice, Step step) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  constexpr int WAVES = THREADS / 64;
  constexpr bool GUMBEL = MODE == CH_GUMBEL, CDF = MODE == CH_CDF;
  static_assert(ONE || !CDF, "slices of the inverse CDF are the greedy choice's");
  __shared__ float red_m[WAVES], red_s[WAVES], red_sum[WAVES];
  __shared__ int first_best, contenders;
  __shared__ double red_steps[WAVES];
  __shared__ Best contender[GUMBEL ? THREADS : 1];
  __shared__ typename std::conditional<CDF, BatchSums<THREADS>, int>::type sums;
  using X = Batch<T, THREADS>;
  const int64_t b = ONE ? blockIdx.x : blockIdx.x / plan.slices;
  const int v0 = ONE ? 0 : static_cast<int>(blockIdx.x % plan.slices) * plan.slice;
  const int v1 = V - v0 < plan.slice ? V : v0 + plan.slice;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const Seen<THREADS> seen(lds, plan);
  const T *row = logits + b * ld;
  X x;
  if (V >= X::N) x.load(row, v0, V);
  const Scale c = row_scale(temp, temp0, b);
  const RowRules r = row_rules(rules, b, V);

  const bool noisy = GUMBEL && c.T > 0.f;
  const float *urow = GUMBEL ? noise_at(noise, rules, b, V) : nullptr;
  Uniforms<T, THREADS, GUMBEL> un;
  if (V >= X::N) un.load(urow, v0, V);
  if (tid == 0) {
    first_best = 0x7fffffff;
    contenders = 0;
  }
  if constexpr (CDF) {
    if (tid < BatchSums<THREADS>::MOST) sums.history[tid] = 0;
    if (tid == 0) {
      sums.walk.found = 0x7fffffff;
      sums.walk.last = -1;
    }
  }
  Mine t;
  // the history's largest logit and its best logit or score of this thread's, apart from the others': what is summed of those
  // does not depend on which thread has which of these
  float hist_m = -FLT_MAX, hist_best = -INFINITY;
  int hist_v = 0x7fffffff;
  if (r.len > 0) {
    seen.fill(r.hist, r.len, v0, v1, plan.slice);
    seen.each([&](int rel, uint32_t &count) {
      const int v = v0 + rel;
      const float z = tame(one_logit(row, r, v, count));
      count = __float_as_uint(z);  // (from here on the token's logit)
      hist_m = vmax2(hist_m, z);
      const float sc = noisy ? gumbel_score(z, urow[v], c) : z;
      if (sc > hist_best || (sc == hist_best && v < hist_v)) {
        hist_best = sc;
        hist_v = v;
      }
    });
  }
  int w = v0;
  [[maybe_unused]] auto keep_sums = [&](int first) {
    if constexpr (CDF)
      if (lane == 0) {
        sums.sum[first / X::TOKENS][wid] = t.sum;
        sums.m[first / X::TOKENS][wid] = t.m;
      }
  };
  for (; w + X::TOKENS < v1; w += X::TOKENS) {
    choose_batch<T, THREADS, MODE, false, true>(x, un, t, row, urow, r, c, seen, v0, w, V);
    keep_sums(w);
  }
  if (w + X::TOKENS <= V)
    choose_batch<T, THREADS, MODE, false, false>(x, un, t, row, urow, r, c, seen, v0, w, V);
  else
    choose_batch<T, THREADS, MODE, true, false>(x, un, t, row, urow, r, c, seen, v0, w, V);
  keep_sums(w);
  const float wm = wave_max_of(vmax2(t.m, hist_m)), wb = wave_max_of(vmax2(t.best, hist_best));
  if (lane == 0) {
    red_m[wid] = wm;
    red_s[wid] = wb;
  }
  __syncthreads();
  float M = red_m[0], most = red_s[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) {
    M = vmax2(M, red_m[i]);
    most = vmax2(most, red_s[i]);
  }
  if constexpr (!CDF) {
    const float ws = wave_sum(t.sum * __builtin_amdgcn_exp2f((t.m - M) * c.L));
    if (lane == 0) red_sum[wid] = ws;
    double steps = 0.;
    if (r.len > 0) {
      seen.each([&](int, uint32_t z) { steps += weight_steps(__uint_as_float(z), M, c); });
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) steps += __shfl_xor(steps, o, 64);
    }
    if (lane == 0) red_steps[wid] = steps;
  }
  if (!noisy) {
    if (most > -INFINITY && t.best == most) atomicMin(&first_best, t.v);
    if (most > -INFINITY && hist_best == most) atomicMin(&first_best, hist_v);
  } else {
    const bool below = most == -INFINITY;  // (t.sum > 0: some logit is finite)
    const auto near = [&](float s) { return s == most || !(s < contender_from(most)); };
    const bool mine = below ? t.sum > 0.f : t.best > -INFINITY && near(t.best);
    const bool hist = r.len > 0 && (below || (hist_best > -INFINITY && near(hist_best)));
    if (mine || hist) {
      Part p = no_part();
      auto offer = [&](int v, float z) {
        Part e = no_part();
        e.z = z;
        e.u = urow[v];
        e.s = gumbel_score(e.z, e.u, c);
        e.v = e.z == -INFINITY ? -1 : v;
        if (better<true>(p, e, c.T)) p = e;
      };
      if (mine && (below || near(t.second))) {
        for (int i = v0; i < v1; i += X::STEP)
          for (int k = 0; k < X::N; ++k) {
            const int v = i + tid * X::N + k;
            if (v < v1 && !(r.len > 0 && seen.has(v - v0))) offer(v, tame(one_logit(row, r, v, 0)));
          }
      } else if (mine) {
        offer(t.v, tame(one_logit(row, r, t.v, 0)));
      }
      if (hist) seen.each([&](int rel, uint32_t z) { offer(v0 + rel, __uint_as_float(z)); });
      if (p.v >= 0) contender[atomicAdd(&contenders, 1)] = Best{p.s, p.z, p.u, p.v};
    }
  }
  __syncthreads();
  if constexpr (CDF) {
    Part p = no_part();
    p.m = vmax2(most, -FLT_MAX);
    if (most > -INFINITY) {
      p.z = most;
      p.v = first_best;
    }
    choose_from_sums(sums, x, row, r, c, seen, V, w / X::TOKENS + 1, p, noise_at(noise, rules, b, 1), choice, step, b);
    return;
  }
  if (tid != 0) return;
  Part p = no_part();
  if (noisy) {
    for (int i = 0; i < contenders; ++i) {
      const Best e = contender[i];
      const Part q = {-FLT_MAX, 0.f, e.s, e.z, e.u, e.v};
      if (better<true>(p, q, c.T)) p = q;
    }
  } else if (most > -INFINITY) {
    p.z = most;
    p.v = first_best;
  }
  p.m = M;
  p.sum = red_sum[0];
#pragma unroll
  for (int i = 1; i < WAVES; ++i) p.sum += red_sum[i];
  double steps = 0.;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) steps += red_steps[i];
  p.sum += static_cast<float>(steps / STEPS);
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

// Inverse CDF of a row in slices: one workgroup per sequence finds the slice that u falls into from the slices' sums (64
// bits, every wavefront by itself), then walks that slice in token order. A row with temperature <= 0 takes the greedy
// choice.
template <typename T>
__global__ __launch_bounds__(CH_THREADS) void choose_cdf_kernel(const T *__restrict__ logits, int64_t ld, Rules rules,
                                                                const float *__restrict__ temp, float temp0,
                                                                Noise noise, int V, Plan plan,
                                                                const Part *__restrict__ parts,
                                                                Choice choice, Step step) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  __shared__ Walk<CH_THREADS> walk;
  using X = Batch<T, CH_THREADS>;
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const int slices = plan.slices, slice = plan.slice;
  const Part *mine = parts + b * slices;
  const RowRules r = row_rules(rules, b, V);
  const Scale c = row_scale(temp, temp0, b);
  const float uniform = *noise_at(noise, rules, b, 1);
  if (tid == 0) {
    walk.found = 0x7fffffff;
    walk.last = -1;
  }
  // every wavefront joins the slices the same way
  Part p = no_part();
  for (int s = lane; s < slices; s += 64) join_parts<false>(p, mine[s], c.L, c.T);
  join_lanes<false>(p, c.L, c.T);
  if (p.v < 0 || !(c.T > 0.f)) {
    if (tid == 0) finish_row(choice, step, b, V, p.v, logp_of(p.z, p, c));
    return;
  }
  auto weight = [&](int s) {
    return s < slices ? static_cast<double>(mine[s].sum * __builtin_amdgcn_exp2f((mine[s].m - p.m) * c.L)) : 0.;
  };
  auto scan = [&](double v) {  // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double up = __shfl_up(v, o, 64);
      if (lane >= o) v += up;
    }
    return v;
  };
  double total = 0.;
  for (int s0 = 0; s0 < slices; s0 += 64) total += __shfl(scan(weight(s0 + lane)), 63, 64);
  const double target = static_cast<double>(uniform) * total;
  // the slice: the first whose running sum passes the target (rounding, or a uniform of 1: the last with any weight)
  int at = 0;
  double before = 0., run = 0.;
  for (int s0 = 0; s0 < slices; s0 += 64) {
    const double v = weight(s0 + lane), upto = scan(v);
    const uint64_t filled = __ballot(v > 0.), past = __ballot(v > 0. && target < before + upto);
    const int l = past != 0 ? __builtin_ctzll(past) : 63 - __builtin_clzll(filled | 1);
    if (filled != 0) {
      at = s0 + l;
      run = before + __shfl(upto - v, l, 64);
    }
    if (past != 0) break;
    before += __shfl(upto, 63, 64);
  }
  const int v0 = at * slice, v1 = V - v0 < slice ? V : v0 + slice;
  const Seen<CH_THREADS> seen(lds, plan);
  const T *row = logits + b * ld;
  X x;
  if (V >= X::N) x.load(row, v0, V);
  if (r.len > 0) {
    seen.fill(r.hist, r.len, v0, v1, slice);
    logits_for_counts(seen, row, r, v0);
  }
  __syncthreads();
  for (int w = v0; w < v1; w += X::TOKENS) {
    if (w > v0 && V >= X::N) x.load(row, w, V);
    walk_batch(x, row, r, c, seen, v0, w, V, p.m, target, run, walk);
    if (walk.found != 0x7fffffff) break;
  }
  if (tid == 0) finish_walk(walk, row, r, c, seen, v0, V, p, choice, step, b);
}

// How B rows of V tokens are cut: about two workgroups per CU in all, of 4096 tokens (one batch) to CH_SLICE. `whole`: one
// workgroup of CH_THREADS_ONE may take a sequence's whole vocabulary, where that spares the slices' joining (CH_SMALL) or
// the sequences load the CUs evenly, to three quarters at least. fp32, 87383 tokens, whole and in slices, us, greedy, Gumbel,
// inverse CDF: 130 sequences 22.1 and 21.4, 36.9 and 34.6, 34.0 and 39.0; 192: 22.8, 27.9; 38.6, 43.6; 34.7, 45.4; 250: 23.8,
// 32.2; 40.3, 51.0; 35.8, 50.4; 300: 38.0, 37.1; 60.4, 58.9; 51.4, 54.4; 400: 39.8, 44.7; 63.8, 72.9; 53.1, 61.6; 512: 43.4,
// 52.9; 69.7, 88.3; 55.4, 70.0. hist_cols: 0 without a history.
static Plan make_plan(int64_t B, int V, int64_t hist_cols, bool whole) {
  constexpr int UNIT = Batch<float, CH_THREADS>::TOKENS;
  static_assert(UNIT == Batch<bf16_t, CH_THREADS>::TOKENS && CH_SLICE % UNIT == 0, "slices are whole batches");
  Plan p = {};
  p.hashed = hist_cols <= CH_HASH_MAX;
  const int64_t cus = device_cus_cached(), units = (static_cast<int64_t>(V) + UNIT - 1) / UNIT;
  const int64_t want = (2 * cus + B - 1) / B, least = (V + CH_SLICE - 1) / CH_SLICE;
  int64_t s = units < want ? units : want;
  if (s < least) s = least;
  int64_t len = (units + s - 1) / s * UNIT;
  p.slices = static_cast<int>((V + len - 1) / len);
  const int64_t rounds = (B + cus - 1) / cus;  // workgroups of the busiest CU, one a sequence
  const bool even = V <= CH_WHOLE && 4 * B >= 3 * rounds * cus;
  if (whole && (p.slices == 1 || (p.hashed && (V <= CH_SMALL || even)))) {
    constexpr int ONE_UNIT = Batch<float, CH_THREADS_ONE>::TOKENS;
    p.one = true;
    p.slices = 1;
    len = (static_cast<int64_t>(V) + ONE_UNIT - 1) / ONE_UNIT * ONE_UNIT;
  }
  p.slice = static_cast<int>(len);
  p.slots = p.slice;
  if (p.hashed)
    for (p.slots = 64; p.slots < 2 * hist_cols;) p.slots *= 2;
  p.listed = (static_cast<int>(hist_cols < p.slice ? hist_cols : p.slice) + 7) & ~7;
  return p;
}

static size_t plan_lds(const Plan &p, bool hist) {
  return hist ? static_cast<size_t>(p.slice) / 8 + static_cast<size_t>(p.slots) * (p.hashed ? 8 : 4) + 16 + 2 * p.listed : 0;
}

// Workgroups of 256 threads that one launch may have (2^32 threads in all).
constexpr int64_t CH_GRID_MAX = int64_t(1) << 24;

static int check_grid(const Plan &p, int64_t B, const char *what) {
  VK_CHECK_ARG(B * p.slices < CH_GRID_MAX, "%s: too many logits for one call", what);
  return VK_OK;
}

static int check_rules(const Rules &r, int64_t B, int V, const char *what) {
  VK_CHECK_ARG(r.hist == nullptr || (r.len != nullptr || r.pos != nullptr), "%s: a history needs lengths", what);
  VK_CHECK_ARG(r.hist == nullptr || (r.hist_cols >= 0 && r.hist_cols <= CH_HIST_MAX && r.hist_ld >= r.hist_cols),
               "%s: histories of at most %d tokens", what, CH_HIST_MAX);
  VK_CHECK_ARG(r.hist == nullptr || r.rep != nullptr || r.rep0 > 0.f, "%s: the repetition penalty must be positive", what);
  VK_CHECK_ARG(r.bias == nullptr || r.bias_ld == 0 || r.bias_ld >= V, "%s: bias row stride below V", what);
  VK_CHECK_ARG(r.allowed == nullptr || (r.n_allowed > 0 && r.allowed_ld >= (V + 31) / 32),
               "%s: masks are rows of ceil(V / 32) words", what);
  VK_CHECK_ARG(r.allowed == nullptr || r.arow != nullptr || r.token_row != nullptr || r.n_allowed == 1 || r.n_allowed == B ||
                   B == 0,
               "%s: masks without row numbers: 1 row or one per sequence", what);
  return VK_OK;
}

static int check_logits(const void *logits, int32_t dtype, int64_t ld, int64_t B, int32_t V, const char *what) {
  VK_CHECK_ARG(B >= 0 && V > 0 && V <= CH_V_MAX && ld >= V, "%s: bad sizes", what);
  VK_CHECK_ARG(B < (int64_t(1) << 20), "%s: at most 2^20 - 1 sequences", what);
  VK_CHECK_ARG(dtype == VK_DTYPE_BF16 || dtype == VK_DTYPE_F32, "%s: logits bf16 or fp32", what);
  VK_CHECK_ARG(B == 0 || logits != nullptr, "%s: null pointer", what);
  return VK_OK;
}

template <typename T>
static int launch_choose(const void *logits, int64_t ld, const Rules &r, const float *temp, float temp0, int mode,
                         const Noise &noise, int64_t B, int V, const Plan &plan, Part *parts, const Choice &choice,
                         const Step &step, hipStream_t s) {
  const T *x = static_cast<const T *>(logits);
  const size_t lds = plan_lds(plan, r.hist != nullptr);
  const unsigned grid = static_cast<unsigned>(B * plan.slices), join = static_cast<unsigned>((B + 3) / 4);
#define VK_SLICES(THREADS, MODE, ONE)                                                                                   \
  choose_slices_kernel<T, THREADS, MODE, ONE><<<grid, THREADS, lds, s>>>(x, ld, r, temp, temp0, noise, V, plan, parts, \
                                                                           choice, step)
  if (plan.one) {
    if (mode == CH_GUMBEL)
      VK_SLICES(CH_THREADS_ONE, CH_GUMBEL, true);
    else if (mode == CH_CDF)
      VK_SLICES(CH_THREADS_ONE, CH_CDF, true);
    else
      VK_SLICES(CH_THREADS_ONE, CH_GREEDY, true);
  } else if (mode == CH_GUMBEL) {
    VK_SLICES(CH_THREADS, CH_GUMBEL, false);
    choose_join_kernel<true><<<join, 256, 0, s>>>(parts, temp, temp0, B, V, plan.slices, choice, step);
  } else {
    VK_SLICES(CH_THREADS, CH_GREEDY, false);
    if (mode == CH_CDF)
      choose_cdf_kernel<T><<<static_cast<unsigned>(B), CH_THREADS, lds, s>>>(x, ld, r, temp, temp0, noise, V, plan, parts,
                                                                             choice, step);
    else
      choose_join_kernel<false><<<join, 256, 0, s>>>(parts, temp, temp0, B, V, plan.slices, choice, step);
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
  const Plan plan = make_plan(B, V, hist ? hist_cols : 0, false);
  rc = check_grid(plan, B, "process_logits");
  if (rc != VK_OK) return rc;
  const size_t lds = plan_lds(plan, hist != nullptr);
  const unsigned grid = static_cast<unsigned>(B * plan.slices);
  hipStream_t s = VK_STREAM(stream);
  const bool lf = dtype == VK_DTYPE_F32, of = out_dtype == VK_DTYPE_F32;
#define VK_PROCESS(T, OT)                                                                                              \
  process_logits_kernel<T, OT><<<grid, CH_THREADS, lds, s>>>(static_cast<const T *>(logits), ld, r, V, plan,            \
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

// Whether a call joins slices, and so needs their results kept.
static int64_t parts_bytes(const Plan &p, int64_t B) {
  return p.one ? 0 : B * p.slices * static_cast<int64_t>(sizeof(Part));
}

extern "C" int vk_choose_tokens_workspace(int64_t B, int32_t V, int64_t hist_cols, int64_t *bytes) {
  VK_CHECK_ARG(bytes && B >= 0 && V > 0 && V <= CH_V_MAX && hist_cols >= 0, "choose_tokens_workspace: bad arguments");
  *bytes = B == 0 ? 0 : parts_bytes(make_plan(B, V, hist_cols, true), B);
  return VK_OK;
}

static int choose(const void *logits, int32_t dtype, int64_t ld, const Rules &r, const float *temp, float temp0,
                  int32_t mode, const Noise &noise, const Choice &choice, const Step &step, int64_t B, int32_t V,
                  void *workspace, int64_t workspace_bytes, void *stream, const char *what) {
  int rc = check_logits(logits, dtype, ld, B, V, what);
  if (rc != VK_OK) return rc;
  rc = check_rules(r, B, V, what);
  if (rc != VK_OK) return rc;
  VK_CHECK_ARG(mode == CH_GREEDY || mode == CH_GUMBEL || mode == CH_CDF,
               "%s: mode 0 (greedy), 1 (Gumbel) or 2 (inverse CDF)", what);
  const int64_t per = mode == CH_GUMBEL ? V : 1;
  VK_CHECK_ARG(mode == CH_GREEDY || ((B == 0 || noise.u != nullptr) && noise.cols > 0 && noise.ld >= noise.cols * per),
               "%s: sampling needs uniforms, rows of columns x %lld", what, static_cast<long long>(per));
  if (B == 0) return VK_OK;
  const Plan plan = make_plan(B, V, r.hist ? r.hist_cols : 0, true);
  rc = check_grid(plan, B, what);
  if (rc != VK_OK) return rc;
  const int64_t need = parts_bytes(plan, B);
  VK_CHECK_ARG(need == 0 || (workspace && vk_aligned16(workspace) && workspace_bytes >= need),
               "%s: a 16-byte aligned workspace of %lld bytes needed", what, static_cast<long long>(need));
  Part *parts = static_cast<Part *>(workspace);
  return dtype == VK_DTYPE_F32 ? launch_choose<float>(logits, ld, r, temp, temp0, mode, noise, B, V, plan, parts, choice,
                                                      step, VK_STREAM(stream))
                               : launch_choose<bf16_t>(logits, ld, r, temp, temp0, mode, noise, B, V, plan, parts, choice,
                                                       step, VK_STREAM(stream));
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
  VK_CHECK_ARG(bias && is_tail && is_homo && (B == 0 || (tok && pos && out)), "choose_update: null pointer");
  VK_CHECK_ARG(homo_stop <= 0 || run != nullptr || B == 0, "choose_update: homopolymer rule needs run");
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
