// Objectives on the decoder's logits and their gradients: the clipped policy loss per token with a KL term, the loss of
// paired log ratios, the divergence from a teacher's list of top logits.
//
// All three are sums over tokens whose gradient by a token's V logits z is, with p = softmax(z / tau),
//   policy, preference   c (onehot(y) - p)                     (tau = 1)
//   distillation         c (Q p_v - sum over the list's entries with id v of their weights), Q = the list's mass
// with one number c per token. Bound by memory: the logits have to be read and their gradients written, 4 or 8 bytes an
// element together, with two exponentials between. So a row is read once, stays in the registers of a group of threads
// (16 lanes to a whole workgroup, by its length) through its maximum, its sum and its gradient, and the few elements that
// differ from c' p_v are written by themselves afterwards. Rows that count nothing are not read.
//
// Exponentials are fp32 (each off by 2e-7 at temperature 1, for distillation by up to 1e-6 far below the top); their sums,
// the logarithm, log-ratios, objectives and sums over tokens are 64 bits. The gradient is rounded once, to the logits' type.
// Every sum runs in a fixed order, which a row's address modulo 16 bytes is part of.
//
// What it reaches, of the 5.2 TB/s that a copy does: fp32 rows of 2500 to 45000 logits 4.5 to 5.3 (policy), 4.5 to 4.9
// (distillation, lists of 32), bf16 rows 4.2 to 4.4 and 3.6 to 4.0 (their exponentials are computed twice past 6 vectors a lane,
// and half the time is VALU issue); rows of 343 bf16 2.5 (the 64-bit numbers of a token, four to a wavefront); the preference
// loss, which has to read its logits twice, 3.1 to 3.8.
#include "common.h"
#include "vocab_rows.h"

namespace vk {

constexpr int OBJ_BLOCKS = 2048;  // most workgroups of a pass over the rows: one partial sum of the loss each
constexpr int OBJ_PARTS = 256;    // partial sums of the tokens' weights

// (temperature 1)
constexpr UnitScale kUnit = {};

struct LogitRows {
  const void *logits;
  int64_t ld_b, ld_t;  // elements from sequence to sequence, token to token
  int64_t N;           // B * T
  uint32_t T;
  int V;
  template <typename T_>
  __device__ __forceinline__ const T_ *row(uint32_t b, uint32_t t) const {
    return static_cast<const T_ *>(logits) + b * ld_b + t * ld_t;
  }
};

// The upstream gradient: a factor of the gradient, and whether there is anything to do (unless_one: the gradient for a
// factor of 1 is there already).
struct Upstream {
  const float *factor;
  int unless_one;
  __device__ __forceinline__ float get() const { return factor ? *factor : 1.f; }
  __device__ __forceinline__ bool done(float f) const { return unless_one && f == 1.f; }
};

// Sum over a workgroup, in a fixed order; every thread gets it. sh: a number per wavefront.
template <int THREADS = 256>
__device__ __forceinline__ double block_sum64(double v, double *sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) v += sh[w];
  return v;
}

// Sum of OBJ_PARTS partial sums by the first wavefront of a workgroup, to *out in shared memory (a barrier has to follow).
__device__ __forceinline__ void sum_parts(const double *parts, double *out) {
  if (threadIdx.x < 64) {
    double v = (parts[threadIdx.x] + parts[threadIdx.x + 64]) + (parts[threadIdx.x + 128] + parts[threadIdx.x + 192]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    if (threadIdx.x == 0) *out = v;
  }
}

// Whether a token counts: masked in, with a target of the vocabulary.
__device__ __forceinline__ bool counts(const uint8_t *mask, const int64_t *targets, int64_t row, int V, int &y) {
  const int64_t t = targets[row];
  y = static_cast<int>(t);
  return mask[row] != 0 && t >= 0 && t < V;
}

// The sum of a row's exponentials without its target's: 1 - p_y = that over s, which keeps its 32 bits where p_y is next to 1
// (c - c p_y is off by 2e-7 c there).
__device__ __forceinline__ float beyond_target(double s, float zy, float top) {
  return static_cast<float>(s - static_cast<double>(exp_of(zy, top, kUnit)));
}

// A token's target and mask as loaded, ahead of their use.
struct Token {
  int64_t target;
  uint8_t mask;
  __device__ __forceinline__ void load(const uint8_t *m, const int64_t *t, int64_t row, int64_t N) {
    const int64_t at = row < N ? row : N - 1;
    target = t[at];
    mask = m[at];
  }
  __device__ __forceinline__ bool counts(int V) const { return mask != 0 && target >= 0 && target < V; }
};

// The same by the rows' own kernels, where that is the cheaper way (count_here below): the tokens of a sequence that count, by
// a group.
template <int GL>
__device__ __forceinline__ int count_sequence(const uint8_t *mask, const int64_t *targets, int64_t b, int64_t T, int V, int lane,
                                              float *sh) {
  int n = 0, y;
  for (int64_t t = lane; t < T; t += GL) n += counts(mask, targets, b * T + t, V, y);
  return static_cast<int>(group_add<GL>(static_cast<float>(n), sh));  // (below 2^24: exact)
}
// All tokens that count or, where weights are given, their sum, by a workgroup; every thread gets it.
template <int THREADS>
__device__ __forceinline__ double count_all(const uint8_t *mask, const int64_t *targets, const float *weights, int64_t N, int V,
                                            double *sh) {
  double v = 0.0;
  int y;
  for (int64_t i = threadIdx.x; i < N; i += THREADS) {
    if (weights) {
      const float w = weights[i];
      if (w > 0.f) v += static_cast<double>(w);
    } else if (counts(mask, targets, i, V, y)) {
      v += 1.0;
    }
  }
  return block_sum64<THREADS>(v, sh);
}

// A wavefront per sequence: how many of its tokens count.
__global__ __launch_bounds__(256) void sequence_counts_kernel(const uint8_t *__restrict__ mask,
                                                             const int64_t *__restrict__ targets, int32_t *__restrict__ out,
                                                             int64_t B, int64_t T, int V, Upstream up) {
  if (up.done(up.get())) return;
  const int64_t b = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (b >= B) return;
  int n = 0, y;
  for (int64_t t = threadIdx.x & 63; t < T; t += 64) n += counts(mask, targets, b * T + t, V, y);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, kWave);
  if ((threadIdx.x & 63) == 0) out[b] = n;
}

// OBJ_PARTS workgroups: partial sums of the tokens that count (targets given) or of the positive weights.
__global__ __launch_bounds__(256) void weight_parts_kernel(const uint8_t *__restrict__ mask,
                                                          const int64_t *__restrict__ targets,
                                                          const float *__restrict__ weights, double *__restrict__ parts,
                                                          int64_t N, int V, Upstream up) {
  __shared__ double sh[4];
  if (up.done(up.get())) return;
  double v = 0.0;
  int y;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < N; i += OBJ_PARTS * 256) {
    if (weights) {
      const float w = weights[i];
      if (w > 0.f) v += static_cast<double>(w);
    } else if (counts(mask, targets, i, V, y)) {
      v += 1.0;
    }
  }
  v = block_sum64(v, sh);
  if (threadIdx.x == 0) parts[blockIdx.x] = v;
}

// loss = the sum of n partial sums
__global__ __launch_bounds__(256) void loss_join_kernel(const double *__restrict__ parts, int n, float *__restrict__ loss) {
  __shared__ double sh[4];
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) v += parts[i];
  v = block_sum64(v, sh);
  if (threadIdx.x == 0) loss[0] = static_cast<float>(v);
}

// ---- the policy loss ----------------------------------------------------------------------------------------------------

struct PolicyArgs {
  const int64_t *targets;
  const uint8_t *mask;
  const float *old_lp, *adv, *ref_lp;
  int adv_per_token;
  double lo, hi, kl_coef;  // the clip's borders 1 - eps_lo, 1 + eps_hi
  int per;                 // VK_PER_*
  double inv_n;
  const int32_t *counts;
  const double *weight_parts;  // NULL: counted here
  float *pg, *kl, *lp;
  void *dlogits;
  double *loss_parts;
  Upstream up;
};

struct PolicyTerms {
  double pg, kl, lp, loss;
  float g;  // the loss's derivative by lp
};
__device__ __forceinline__ PolicyTerms policy_terms(double lp, float old_lp, float adv, bool has_ref, float ref_lp, double lo,
                                                    double hi, double kl_coef) {
  PolicyTerms t;
  t.lp = lp;
  const double d = lp - static_cast<double>(old_lp), A = static_cast<double>(adv);
  const double r = exp_64(d);
  const double cut = r < lo ? lo : r > hi ? hi : r;
  const double a1 = r * A, a2 = cut * A;
  const double inner = (r >= lo && r <= hi) ? A : 0.0;
  const double slope = a1 < a2 ? A : a2 < a1 ? inner : 0.5 * (A + inner);  // equal sides share evenly
  t.pg = -(a1 < a2 ? a1 : a2);
  if (!(a1 < a2) && !(a2 <= a1)) t.pg = a1 + a2;  // (a NaN among them)
  double g = -slope * r;
  t.kl = 0.0;
  t.loss = t.pg;
  if (has_ref) {
    const double x = static_cast<double>(ref_lp) - lp;
    t.kl = exp_beyond_line(x);
    if (kl_coef != 0.0) {
      t.loss += kl_coef * t.kl;
      g -= kl_coef * (x < -40.0 ? -1.0 : t.kl + x);  // (exp(x) - 1: of -inf too)
    }
  }
  t.g = static_cast<float>(g);
  return t;
}

// COUNTS: each group counts its rows' sequences (per sequence, where no launch did).
template <typename Row, bool COUNTS>
__global__ __launch_bounds__(group_threads(Row::GL), Row::WAVES_A_SIMD) void policy_rows_kernel(LogitRows in, PolicyArgs a) {
  typedef typename Row::type T;
  constexpr int GL = Row::GL, GROUPS = group_threads(GL) / GL;
  __shared__ RowSums<GL> sh;
  __shared__ float count_sh[COUNTS && GL > 64 ? GL / 64 : 1];
  __shared__ float coef_sh;
  __shared__ double total_sh, loss_sh[group_threads(GL) / 64];
  const float factor = a.up.get();
  if (a.up.done(factor)) return;
  const int lane = lane_of<GL>(), group = group_of<GL>();
  double w_all = a.inv_n;
  if (a.per == VK_PER_TOKEN_MEAN) {
    double total;
    if (a.weight_parts) {
      sum_parts(a.weight_parts, &total_sh);
      __syncthreads();
      total = total_sh;
    } else {
      total = count_all<group_threads(GL)>(a.mask, a.targets, nullptr, in.N, in.V, loss_sh);
    }
    w_all = 1.0 / fmax(total, 1.0);
  }
  double loss = 0.0;
  int turn = 0;  // a workgroup's wavefronts do the tokens' 64-bit numbers in turn: they are on one SIMD each
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group;
  for (; row < in.N; row += step) {
    Token token;
    token.load(a.mask, a.targets, row, in.N);
    const uint32_t b = static_cast<uint32_t>(row) / in.T, t = static_cast<uint32_t>(row) % in.T;
    T *d = a.dlogits ? static_cast<T *>(a.dlogits) + row * in.V : nullptr;
    const int lead = GL > 64 ? turn : 0;
    if (GL > 64) turn = (turn + 64) % GL;
    if (!token.counts(in.V)) {
      if (d) Row::zero(d, in.V, lane);
      if (lane == 0) {
        if (a.lp) a.lp[row] = 0.f;
        if (a.pg) a.pg[row] = 0.f;
        if (a.kl) a.kl[row] = 0.f;
      }
      continue;
    }
    const T *z = in.row<T>(b, t);
    const int y = static_cast<int>(token.target);
    const float zy = load_one(z + y);
    Row r;
    r.load(z, in.V, lane);
    int among = 1;
    if constexpr (COUNTS) among = count_sequence<GL>(a.mask, a.targets, b, in.T, in.V, lane, count_sh);
    float top;
    double s;
    row_stats<GL>(r, kUnit, sh, top, s);
    float c = 0.f;
    if (GL <= 64 || lane == lead) {
      const double lp = static_cast<double>(zy) - static_cast<double>(top) - log_of(s);
      const PolicyTerms p = policy_terms(lp, a.old_lp[row], a.adv[a.adv_per_token ? row : b], a.ref_lp != nullptr,
                                         a.ref_lp ? a.ref_lp[row] : 0.f, a.lo, a.hi, a.kl_coef);
      if (!COUNTS && a.per == VK_PER_SEQUENCE) among = a.counts[b];
      const double w = w_all / static_cast<double>(among);
      c = static_cast<float>(w * static_cast<double>(p.g) * static_cast<double>(factor));
      if (lane == lead) {
        loss += w * p.loss;
        if (a.lp) a.lp[row] = static_cast<float>(p.lp);
        if (a.pg) a.pg[row] = static_cast<float>(p.pg);
        if (a.kl) a.kl[row] = static_cast<float>(p.kl);
      }
      if (GL > 64) coef_sh = c;
    }
    if (!d) {
      group_sync<GL>();
      continue;
    }
    if constexpr (GL > 64) {
      __syncthreads();
      c = coef_sh;
    }
    const float k = -c / static_cast<float>(s);
    const float rest = beyond_target(s, zy, top);
    r.write(d, lane, top, kUnit, k);
    // (after this thread's own vector that holds it)
    if (lane == owner_of<T, GL>(r.s, y)) store_one(d + y, -k * rest);
  }
  if (!a.loss_parts) return;
  loss = block_sum64<group_threads(GL)>(loss, loss_sh);
  if (threadIdx.x == 0) a.loss_parts[blockIdx.x] = loss;
}

// ---- paired log ratios --------------------------------------------------------------------------------------------------

struct RowStats {
  float top, rs, rest;  // a row's maximum, one over its sum of exponentials, that sum without its target's
};

struct PairArgs {
  const int64_t *targets;
  const uint8_t *mask;
  const float *ref_lp;
  float *lp;
  double *ratio;
  RowStats *stats;
};

// Each token's log-probability, its log-ratio and what its gradient will need.
template <typename Row>
__global__ __launch_bounds__(group_threads(Row::GL), Row::RATIO_WAVES) void token_ratio_kernel(LogitRows in, PairArgs a) {
  typedef typename Row::type T;
  constexpr int GL = Row::GL, GROUPS = group_threads(GL) / GL;
  __shared__ RowSums<GL> sh;
  const int lane = lane_of<GL>(), group = group_of<GL>();
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group;
  Token next;
  next.load(a.mask, a.targets, row, in.N);
  for (; row < in.N; row += step) {
    const Token token = next;
    next.load(a.mask, a.targets, row + step, in.N);
    const uint32_t b = static_cast<uint32_t>(row) / in.T, t = static_cast<uint32_t>(row) % in.T;
    if (!token.counts(in.V)) {
      if (lane == 0) {
        a.lp[row] = 0.f;
        a.ratio[row] = 0.0;
      }
      continue;
    }
    const T *z = in.row<T>(b, t);
    const float zy = load_one(z + static_cast<int>(token.target)), ref_lp = a.ref_lp ? a.ref_lp[row] : 0.f;
    Row r;
    r.load(z, in.V, lane);
    float top;
    double s;
    row_stats<GL>(r, kUnit, sh, top, s);
    if (lane == 0) {
      const double lp = static_cast<double>(zy) - static_cast<double>(top) - log_called(s);
      a.lp[row] = static_cast<float>(lp);
      a.ratio[row] = lp - static_cast<double>(ref_lp);
      if (a.stats) a.stats[row] = RowStats{top, 1.f / static_cast<float>(s), beyond_target(s, zy, top)};
    }
  }
}

// A workgroup per sequence: its log-ratio over all tokens that count, over its length where one is given.
__global__ __launch_bounds__(256) void sequence_ratio_kernel(const double *__restrict__ ratio,
                                                            const float *__restrict__ lengths, double *__restrict__ out,
                                                            int64_t T) {
  __shared__ double sh[4];
  const int64_t b = blockIdx.x;
  double v = 0.0;
  for (int64_t t = threadIdx.x; t < T; t += 256) v += ratio[b * T + t];
  v = block_sum64(v, sh);
  if (threadIdx.x == 0) out[b] = lengths ? v / static_cast<double>(lengths[b]) : v;
}

// log(1 + exp(x))
__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

__device__ __forceinline__ double logistic(double x) {
  const double e = exp(-fabs(x));
  return (x >= 0.0 ? 1.0 : e) / (1.0 + e);
}

// Pair p's margin, the loss's derivative by its log-ratio difference, and (returned) its share of the loss over inv_n.
__device__ __forceinline__ double pair_terms(const double *ratio, const int64_t *pairs, int64_t p, int64_t B, double beta,
                                             double target, double smoothing, double inv_n, float *margin, double *slope) {
  const int64_t c = pairs ? pairs[2 * p] : 2 * p, r = pairs ? pairs[2 * p + 1] : 2 * p + 1;
  double h = 0.0, dh = 0.0, loss = 0.0;
  if (c >= 0 && c < B && r >= 0 && r < B) {
    h = beta * (ratio[c] - ratio[r]) - target;
    // (a side without weight is left out: the margin may be infinite)
    loss = (smoothing < 1.0 ? (1.0 - smoothing) * softplus(-h) : 0.0) + (smoothing > 0.0 ? smoothing * softplus(h) : 0.0);
    // sigma(h) - (1 - smoothing), without cancellation where the margin is far
    dh = inv_n * beta * (smoothing * logistic(h) - (1.0 - smoothing) * logistic(-h));
  }
  margin[p] = static_cast<float>(h);
  slope[p] = dh;
  return loss;
}

// The derivative of the loss by the tokens' log-probabilities of sequence b, from all pairs that name it, by a wavefront: each
// sequence looks at every pair, and one workgroup has the pairs' own numbers. For up to some thousand pairs: 512 sequences with
// 1024, 8192, 65536 and 2^20 of them, 28, 72, 490 and 8350 us a call of short rows.
__device__ __forceinline__ double sequence_slope(const double *slope, const int64_t *pairs, int64_t b, int64_t P, int lane) {
  if (!pairs) return b / 2 < P ? ((b & 1) ? -slope[b / 2] : slope[b / 2]) : 0.0;
  double v = 0.0;
  for (int64_t p = lane; p < P; p += 64) {
    const int64_t c = pairs[2 * p], r = pairs[2 * p + 1];
    const double s = slope[p];
    if (c == b) v += s;
    if (r == b) v -= s;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

// One workgroup: every pair's margin and slope, and the loss.
__global__ __launch_bounds__(256) void pair_loss_kernel(const double *__restrict__ ratio, const int64_t *__restrict__ pairs,
                                                       int64_t P, int64_t B, double beta, double target, double smoothing,
                                                       double inv_n, float *__restrict__ margin, double *__restrict__ slope,
                                                       float *__restrict__ loss) {
  __shared__ double sh[4];
  double sum = 0.0;
  for (int64_t p = threadIdx.x; p < P; p += 256)
    sum += pair_terms(ratio, pairs, p, B, beta, target, smoothing, inv_n, margin, slope);
  sum = block_sum64(sum, sh);
  if (threadIdx.x == 0) loss[0] = static_cast<float>(sum * inv_n);
}

// A wavefront per sequence.
__global__ __launch_bounds__(256) void sequence_slope_kernel(const double *__restrict__ slope, const int64_t *__restrict__ pairs,
                                                            const float *__restrict__ lengths, int64_t P, int64_t B,
                                                            float *__restrict__ coef) {
  const int64_t b = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (b >= B) return;
  const double v = sequence_slope(slope, pairs, b, P, threadIdx.x & 63);
  if ((threadIdx.x & 63) == 0) coef[b] = static_cast<float>(lengths ? v / static_cast<double>(lengths[b]) : v);
}

// The three steps above in one workgroup, for calls of few tokens: two launches less. 260 tokens in 2 pairs: 28.1 -> 22.8 us;
// 32 sequences of 147 tokens in 48 pairs take it 7 us, as long as the launches do.
constexpr int64_t PAIRS_AT_ONCE_TOKENS = 8192, PAIRS_AT_ONCE_PAIRS = 1024;
__global__ __launch_bounds__(1024) void pairs_at_once_kernel(const double *__restrict__ token_ratio,
                                                             const float *__restrict__ lengths, const int64_t *__restrict__ pairs,
                                                             int P, int B, int64_t T, double beta, double target,
                                                             double smoothing, double inv_n, double *ratio, double *slope,
                                                             float *__restrict__ margin, float *__restrict__ loss,
                                                             float *__restrict__ coef) {
  __shared__ double sh[16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int b = wave; b < B; b += 16) {
    double v = 0.0;
    for (int64_t t = lane; t < T; t += 64) v += token_ratio[b * T + t];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    if (lane == 0) ratio[b] = lengths ? v / static_cast<double>(lengths[b]) : v;
  }
  __syncthreads();
  double sum = 0.0;
  for (int p = threadIdx.x; p < P; p += 1024)
    sum += pair_terms(ratio, pairs, p, B, beta, target, smoothing, inv_n, margin, slope);
  sum = block_sum64<1024>(sum, sh);
  if (threadIdx.x == 0) loss[0] = static_cast<float>(sum * inv_n);
  for (int b = wave; b < B; b += 16) {
    const double v = sequence_slope(slope, pairs, b, P, lane);
    if (lane == 0) coef[b] = static_cast<float>(lengths ? v / static_cast<double>(lengths[b]) : v);
  }
}

// dlogits = c (onehot(y) - softmax) with the rows' maxima and sums known.
template <typename Row>
__global__ __launch_bounds__(group_threads(Row::GL)) void softmax_grad_kernel(LogitRows in, PairArgs a,
                                                                             const float *__restrict__ coef, void *dlogits,
                                                                             Upstream up) {
  typedef typename Row::type T;
  constexpr int GL = Row::GL, GROUPS = group_threads(GL) / GL;
  const float factor = up.get();
  if (up.done(factor)) return;
  const int lane = lane_of<GL>(), group = group_of<GL>();
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group;
  Token next;
  next.load(a.mask, a.targets, row, in.N);
  for (; row < in.N; row += step) {
    const Token token = next;
    next.load(a.mask, a.targets, row + step, in.N);
    const uint32_t b = static_cast<uint32_t>(row) / in.T, t = static_cast<uint32_t>(row) % in.T;
    T *d = static_cast<T *>(dlogits) + row * in.V;
    const float c = coef[b] * factor;
    if (!token.counts(in.V) || c == 0.f) {
      Row::zero(d, in.V, lane);
      continue;
    }
    const T *z = in.row<T>(b, t);
    const int y = static_cast<int>(token.target);
    const RowStats st = a.stats[row];
    Row r;
    r.load(z, in.V, lane);
    const float k = -c * st.rs;
    r.write_fresh(d, lane, st.top, kUnit, k);
    if (lane == owner_of<T, GL>(r.s, y)) store_one(d + y, -k * st.rest);
  }
}

// ---- distillation -------------------------------------------------------------------------------------------------------

constexpr int LIST_MAX = 128;

struct DistillArgs {
  const void *values;
  int values_bf16;
  const void *ids;
  int ids_64;
  int K;
  const float *t_lse, *weights;
  double tau, inv_tau;
  ExpScale scale;
  int mean;  // the weights over their sum (weight_parts), else times inv_n
  double inv_n;
  const double *weight_parts;  // NULL: summed here
  float *kl;
  void *dlogits;
  double *loss_parts;
  Upstream up;
};

// What the lanes of the list's wavefront (or of a group of 16) hold of it: entry i with lane i % LL.
template <int LL, int LONGEST>
struct TeacherList {
  static constexpr int N = LONGEST < LL ? 1 : LONGEST / LL;
  float q[N];   // the entry's weight, 0 where there is none
  float zt[N];  // the student's logit there
  int id[N];    // -1 where there is none
};

// LONGEST: the longest list. (Rows of 16 lanes hold lists of up to 32 in two entries a lane and longer ones in eight, which
// cost registers: 131072 x 343 bf16, lists of 32: 97 -> 81 us.)
template <typename Row, int LONGEST>
__global__ __launch_bounds__(group_threads(Row::GL), Row::DISTILL_WAVES) void distill_rows_kernel(LogitRows in, DistillArgs a) {
  typedef typename Row::type T;
  constexpr int GL = Row::GL, GROUPS = group_threads(GL) / GL;
  constexpr int LL = GL < 64 ? GL : 64;                       // lanes that hold the list
  constexpr int BITS = GL == 16 ? 1024 : GL == 64 ? 4096 : 65536;  // ids seen, by their low bits
  __shared__ RowSums<GL> sh;
  __shared__ uint32_t seen[GROUPS * BITS / 32];
  __shared__ double total_sh, loss_sh[group_threads(GL) / 64];
  __shared__ float qs[GROUPS][LONGEST];
  __shared__ int ids_sh[GROUPS][LONGEST];
  __shared__ float mass_sh;
  const float factor = a.up.get();
  if (a.up.done(factor)) return;
  const int lane = lane_of<GL>(), group = group_of<GL>();
  for (int i = threadIdx.x; i < GROUPS * BITS / 32; i += group_threads(GL)) seen[i] = 0;
  double w_all = a.inv_n;
  if (a.mean) {
    double total;
    if (a.weight_parts) {
      sum_parts(a.weight_parts, &total_sh);
      __syncthreads();
      total = total_sh;
    } else {
      total = count_all<group_threads(GL)>(nullptr, nullptr, a.weights, in.N, in.V, loss_sh);
    }
    w_all = total > 0.0 ? 1.0 / total : 0.0;
  }
  __syncthreads();  // (what was seen: nothing)
  uint32_t *bits = seen + group * (BITS / 32);
  const ExpScale scale = a.scale;
  double loss = 0.0;
  int turn = 0;  // a workgroup's wavefronts hold the list and do the token's numbers in turn
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group; row < in.N;
       row += static_cast<int64_t>(gridDim.x) * GROUPS) {
    const uint32_t b = static_cast<uint32_t>(row) / in.T, t = static_cast<uint32_t>(row) % in.T;
    T *d = a.dlogits ? static_cast<T *>(a.dlogits) + row * in.V : nullptr;
    const float w = a.weights ? a.weights[row] : 1.f;
    const int ll = GL > 64 ? static_cast<int>(threadIdx.x) - turn : lane;  // the list's lanes: 0 .. LL - 1
    const bool holds = ll >= 0 && ll < LL;
    if (GL > 64) turn = (turn + 64) % GL;
    if (!(w > 0.f)) {
      if (d) Row::zero(d, in.V, lane);
      if (lane == 0 && a.kl) a.kl[row] = 0.f;
      continue;
    }
    const T *z = in.row<T>(b, t);
    Row r;
    r.load(z, in.V, lane);
    // the list, with the group's first lanes: weights q, their sum, and sum q (log q - (z - near) / tau) by its largest student
    // logit, `near` (not by 0: a row masked by the type's lowest value would lose its logarithms beside 1e38)
    TeacherList<LL, LONGEST> list;
    double cross = 0.0, mass64 = 0.0;
    float mass = 0.f, near = -FLT_MAX;
    bool twice = false;
    if (holds) {
      float tv[TeacherList<LL, LONGEST>::N], most = -INFINITY;
#pragma unroll
      for (int i = 0; i < TeacherList<LL, LONGEST>::N; ++i) {
        const int e = i * LL + ll;
        list.id[i] = -1;
        list.zt[i] = 0.f;
        list.q[i] = 0.f;
        tv[i] = -INFINITY;
        if (i * LL >= a.K) continue;  // (the same for all: nothing of it runs for shorter lists)
        if (e >= a.K) continue;
        const int64_t at = row * a.K + e;
        const int64_t id = a.ids_64 ? static_cast<const int64_t *>(a.ids)[at] : static_cast<const int32_t *>(a.ids)[at];
        if (id < 0 || id >= in.V) continue;
        const float x = a.values_bf16 ? load_one(static_cast<const bf16_t *>(a.values) + at)
                                      : static_cast<const float *>(a.values)[at];
        if (x == -INFINITY) continue;
        list.id[i] = static_cast<int>(id);
        list.zt[i] = load_one(z + id);
        tv[i] = x;
        most = fmaxf(most, x);
      }
      // weights q: the entries' exponentials over their sum, or over the teacher's
      const double lse_q = a.t_lse ? static_cast<double>(a.t_lse[row]) : 0.0;
      if (a.t_lse) {
#pragma unroll
        for (int i = 0; i < TeacherList<LL, LONGEST>::N; ++i) {
          if (i * LL >= a.K) break;
          const double x = static_cast<double>(tv[i]) * a.inv_tau - lse_q;
          const float xf = static_cast<float>(x), e = expf(xf);
          // (beyond 32 bits, as the type's lowest value over a small temperature is, the narrowing leaves no remainder)
          const float exact = e > 0.f && e < INFINITY ? fmaf(e, static_cast<float>(x - static_cast<double>(xf)), e) : e;
          list.q[i] = list.id[i] >= 0 ? exact : 0.f;
        }
        most = 0.f;
      } else {
#pragma unroll
        for (int o = LL / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, kWave));
#pragma unroll
        for (int i = 0; i < TeacherList<LL, LONGEST>::N; ++i) {
          if (i * LL >= a.K) break;
          list.q[i] = list.id[i] >= 0 ? exp_of(tv[i], most, scale) : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < TeacherList<LL, LONGEST>::N; ++i) {
        if (i * LL >= a.K) break;
        if (list.q[i] != 0.f) near = fmaxf(near, list.zt[i]);
      }
#pragma unroll
      for (int o = LL / 2; o > 0; o >>= 1) near = fmaxf(near, __shfl_xor(near, o, kWave));
#pragma unroll
      for (int i = 0; i < TeacherList<LL, LONGEST>::N; ++i) {
        if (i * LL >= a.K) break;
        if (list.id[i] < 0) continue;
        mass64 += static_cast<double>(list.q[i]);
        if (list.q[i] != 0.f)
          cross += static_cast<double>(list.q[i]) *
                   (((static_cast<double>(tv[i]) - static_cast<double>(most)) * a.inv_tau - lse_q) -
                    (static_cast<double>(list.zt[i]) - static_cast<double>(near)) * a.inv_tau);
        if (d) {
          const uint32_t bit = 1u << (list.id[i] & 31);
          twice |= (atomicOr(&bits[(list.id[i] & (BITS - 1)) >> 5], bit) & bit) != 0;
        }
      }
#pragma unroll
      for (int o = LL / 2; o > 0; o >>= 1) {
        mass64 += __shfl_xor(mass64, o, kWave);
        cross += __shfl_xor(cross, o, kWave);
        twice |= __shfl_xor(static_cast<int>(twice), o, kWave) != 0;
      }
      mass = static_cast<float>(mass64);
      if (!a.t_lse && mass64 != 0.0) {
        cross = cross / mass64 - log_called(mass64);
        const float rs = static_cast<float>(1.0 / mass64);
#pragma unroll
        for (int i = 0; i < TeacherList<LL, LONGEST>::N; ++i) list.q[i] *= rs;
        mass = mass64 > 0.0 ? 1.f : mass;
        mass64 = mass;
      }
      if (GL > 64 && ll == 0) mass_sh = mass;
      if (twice) {
#pragma unroll
        for (int i = 0; i < TeacherList<LL, LONGEST>::N; ++i) {
          const int e = i * LL + ll;
          if (e < a.K) {
            ids_sh[group][e] = list.id[i];
            qs[group][e] = list.q[i];
          }
        }
      }
    }
    float top;
    double s;
    row_stats<GL>(r, scale, sh, top, s);
    if constexpr (GL > 64) mass = mass_sh;
    const double share = static_cast<double>(w) * w_all * a.tau;
    if (ll == 0) {
      // sum q (log q - log p), log p = (z - top) / tau - log s
      const double kl =
          mass == 0.f ? 0.0
                      : cross + mass64 * ((static_cast<double>(top) - static_cast<double>(near)) * a.inv_tau + log_called(s));
      loss += share * a.tau * kl;
      if (a.kl) a.kl[row] = static_cast<float>(kl);
    }
    if (d) {
      const float c = static_cast<float>(share * static_cast<double>(factor));
      const float k = mass == 0.f ? 0.f : c * mass / static_cast<float>(s);
      if (mass == 0.f)
        Row::zero(d, in.V, lane);
      else
        r.write(d, lane, top, scale, k);
      group_sync<GL>();
      if (holds) {
#pragma unroll
        for (int i = 0; i < TeacherList<LL, LONGEST>::N; ++i) {
          const int id = list.id[i], e = i * LL + ll;
          if (i * LL >= a.K) break;
          if (id < 0) continue;
          float q = list.q[i];
          bool mine = true;
          if (twice) {  // equal ids: the first of them writes their sum
            q = 0.f;
            for (int j = 0; j < a.K; ++j)
              if (ids_sh[group][j] == id) {
                mine &= j >= e;
                q += qs[group][j];
              }
          }
          if (mine && mass != 0.f) store_one(d + id, exp_of(list.zt[i], top, scale) * k - c * q);
          bits[(id & (BITS - 1)) >> 5] = 0;
        }
      }
    }
    group_sync<GL>();  // before the next row's list
  }
  if (!a.loss_parts) return;
  loss = block_sum64<group_threads(GL)>(loss, loss_sh);
  if (threadIdx.x == 0) a.loss_parts[blockIdx.x] = loss;
}

// ---- launches -----------------------------------------------------------------------------------------------------------

// Workgroups of a pass over n rows: all of them, or as many as the chip holds, each walking its share.
inline unsigned row_blocks(int64_t n, int gl) {
  const int threads = group_threads(gl), groups = threads / gl;
  const int64_t want = (n + groups - 1) / groups;
  int64_t most = static_cast<int64_t>(device_cus_cached()) * (2048 / threads);
  if (most > OBJ_BLOCKS) most = OBJ_BLOCKS;
  return static_cast<unsigned>(want < most ? want : most);
}

// Whether the rows' kernel counts the tokens itself: a launch less (2.7 us of the host, 1.6 on the GPU and the gap), for N
// numbers read by every workgroup or T by every row. 148 tokens of 37: 24.0 -> 21.3 us. Calls whose rows are more than the
// chip holds at once keep the launch, which is nothing beside them.
inline bool count_here(int64_t n, int64_t T, int gl, bool per_sequence) {
  return gl > 1 && n <= 2048 && (!per_sequence || T <= 4 * gl);
}

template <typename T, bool LANES, typename F>
int with_form(int V, F f) {
  if constexpr (LANES) {
    if (V <= 8) return f(static_cast<RowLane<T, 8> *>(nullptr));
    if (V <= 16) return f(static_cast<RowLane<T, 16> *>(nullptr));
    if (V <= 32) return f(static_cast<RowLane<T, 32> *>(nullptr));
  }
  return row_form((V + kVec<T> - 1) / kVec<T>, [&](auto gl, auto nv) {
    typedef typename RowForm<T, decltype(gl)::value, decltype(nv)::value>::type Row;
    return f(static_cast<Row *>(nullptr));
  });
}
// LANES: rows of up to 32 logits a thread each
template <bool LANES, typename F>
int with_row(int dtype, int V, F f) {
  return dtype == VK_DTYPE_BF16 ? with_form<bf16_t, LANES>(V, f) : with_form<float, LANES>(V, f);
}

}  // namespace vk

using namespace vk;

namespace {

int check_rows(const char *what, const void *logits, int32_t dtype, int64_t ld_b, int64_t ld_t, int64_t B, int64_t T, int32_t V) {
  VK_CHECK_ARG(dtype == VK_DTYPE_BF16 || dtype == VK_DTYPE_F32, "%s: logits are bf16 or fp32", what);
  VK_CHECK_ARG(B >= 0 && T >= 0 && V > 0 && V <= (1 << 30) && B < (int64_t(1) << 31) && T < (int64_t(1) << 31) &&
                   B * T < (int64_t(1) << 31),
               "%s: bad sizes", what);
  VK_CHECK_ARG(B * T == 0 || logits, "%s: null logits", what);
  VK_CHECK_ARG((T < 2 || ld_t >= V) && (B < 2 || ld_b >= V) && ld_t >= 0 && ld_b >= 0, "%s: rows overlap", what);
  return VK_OK;
}

}  // namespace

extern "C" int vk_objective_workspace(int64_t B, int64_t T, int64_t P, int64_t *bytes) {
  VK_CHECK_ARG(bytes && B >= 0 && T >= 0 && P >= 0 && B < (int64_t(1) << 31) && T < (int64_t(1) << 31) && P < (int64_t(1) << 31) &&
                   B * T < (int64_t(1) << 31),
               "objective_workspace: bad arguments");
  // partial sums of weights and loss, then per sequence a 64-bit and a 32-bit number, per pair a 64-bit one, per token a
  // log-ratio and what the row's gradient needs
  *bytes = 8 * (OBJ_PARTS + OBJ_BLOCKS) + 16 * B + (P > 0 ? 8 * P + 20 * B * T : 0) + 16;
  return VK_OK;
}

extern "C" int vk_policy_score(const void *logits, int32_t dtype, int64_t ld_b, int64_t ld_t, const int64_t *targets,
                               const uint8_t *mask, const float *old_lp, const float *adv, int32_t adv_per_token,
                               const float *ref_lp, double eps_lo, double eps_hi, double kl_coef, int32_t per, double inv_n,
                               float *loss, float *pg, float *kl, float *lp, void *dlogits, const float *upstream,
                               int32_t unless_one, int64_t B, int64_t T, int32_t V, void *ws, int64_t ws_bytes, void *stream) {
  int rc = check_rows("policy_score", logits, dtype, ld_b, ld_t, B, T, V);
  if (rc != VK_OK) return rc;
  VK_CHECK_ARG(per >= VK_PER_SEQUENCE && per <= VK_PER_TOKEN_MEAN, "policy_score: per");
  VK_CHECK_ARG(ref_lp || kl_coef == 0.0, "policy_score: the KL term needs ref_lp");
  VK_CHECK_ARG(!kl || ref_lp, "policy_score: kl needs ref_lp");
  VK_CHECK_ARG(!unless_one || upstream, "policy_score: unless_one needs the upstream gradient");
  int64_t need;
  rc = vk_objective_workspace(B, T, 0, &need);
  if (rc != VK_OK) return rc;
  VK_CHECK_ARG(ws && vk_aligned16(ws) && ws_bytes >= need, "policy_score: the workspace needs %lld bytes", (long long)need);
  const int64_t N = B * T;
  VK_CHECK_ARG(N == 0 || (targets && mask && old_lp && adv), "policy_score: null pointer");
  hipStream_t st = VK_STREAM(stream);
  double *weight_parts = static_cast<double *>(ws), *loss_parts = weight_parts + OBJ_PARTS;
  int32_t *counts = reinterpret_cast<int32_t *>(loss_parts + OBJ_BLOCKS);
  const Upstream up{upstream, unless_one};
  unsigned blocks = 0;
  if (N > 0) {
    const LogitRows in{logits, ld_b, ld_t, N, static_cast<uint32_t>(T), V};
    PolicyArgs a{targets, mask, old_lp, adv, ref_lp, adv_per_token, 1.0 - eps_lo, 1.0 + eps_hi, kl_coef, per, inv_n,
                       counts, weight_parts, pg, kl, lp, dlogits, loss ? loss_parts : nullptr, up};
    rc = with_row<true>(dtype, V, [&](auto *form) {
      typedef typename std::remove_pointer<decltype(form)>::type Row;
      blocks = row_blocks(N, Row::GL);
      if (per != VK_PER_TOKEN && count_here(N, T, Row::GL, per == VK_PER_SEQUENCE)) {
        a.weight_parts = nullptr;
        if (per == VK_PER_SEQUENCE) {
          if constexpr (Row::GL > 1) {
            policy_rows_kernel<Row, true><<<blocks, group_threads(Row::GL), 0, st>>>(in, a);
            return launch_status("policy_score");
          }
        }
      } else if (per == VK_PER_SEQUENCE) {
        sequence_counts_kernel<<<static_cast<unsigned>((B + 3) / 4), 256, 0, st>>>(mask, targets, counts, B, T, V, up);
      } else if (per == VK_PER_TOKEN_MEAN) {
        weight_parts_kernel<<<OBJ_PARTS, 256, 0, st>>>(mask, targets, nullptr, weight_parts, N, V, up);
      }
      const int rc2 = launch_status("policy_score counts");
      if (rc2 != VK_OK) return rc2;
      policy_rows_kernel<Row, false><<<blocks, group_threads(Row::GL), 0, st>>>(in, a);
      return launch_status("policy_score");
    });
    if (rc != VK_OK) return rc;
  }
  if (!loss) return VK_OK;
  loss_join_kernel<<<1, 256, 0, st>>>(loss_parts, static_cast<int>(blocks), loss);
  return launch_status("policy_score loss");
}

extern "C" int vk_preference_score(const void *logits, int32_t dtype, int64_t ld_b, int64_t ld_t, const int64_t *targets,
                                   const uint8_t *mask, const float *ref_lp, const float *lengths, const int64_t *pairs,
                                   int64_t P, double beta, double target, double smoothing, double inv_n, float *loss,
                                   float *margin, float *lp, void *dlogits, const float *upstream, int32_t unless_one,
                                   int32_t parts, int64_t B, int64_t T, int32_t V, void *ws, int64_t ws_bytes, void *stream) {
  int rc = check_rows("preference_score", logits, dtype, ld_b, ld_t, B, T, V);
  if (rc != VK_OK) return rc;
  VK_CHECK_ARG(P >= 0 && (pairs || P == 0 || B == 2 * P), "preference_score: without pairs, sequences 2 p and 2 p + 1 are pair p");
  VK_CHECK_ARG(parts >= 1 && parts <= 3, "preference_score: parts");
  VK_CHECK_ARG(!unless_one || upstream, "preference_score: unless_one needs the upstream gradient");
  int64_t need;
  rc = vk_objective_workspace(B, T, P > 0 ? P : 1, &need);
  if (rc != VK_OK) return rc;
  VK_CHECK_ARG(ws && vk_aligned16(ws) && ws_bytes >= need, "preference_score: the workspace needs %lld bytes",
               (long long)need);
  const int64_t N = B * T;
  VK_CHECK_ARG(N == 0 || (targets && mask), "preference_score: null pointer");
  const bool forward = (parts & 1) != 0, backward = (parts & 2) != 0;
  VK_CHECK_ARG(!forward || (loss && (P == 0 || margin) && (N == 0 || lp)), "preference_score: null output");
  VK_CHECK_ARG(!backward || N == 0 || dlogits, "preference_score: null gradient");
  hipStream_t st = VK_STREAM(stream);
  double *ratio = static_cast<double *>(ws), *slope = ratio + B;
  double *token_ratio = slope + (P > 0 ? P : 1);
  RowStats *stats = reinterpret_cast<RowStats *>(token_ratio + N);
  float *coef = reinterpret_cast<float *>(stats + N);
  const LogitRows in{logits, ld_b, ld_t, N, static_cast<uint32_t>(T), V};
  const PairArgs a{targets, mask, ref_lp, lp, token_ratio, stats};
  if (forward) {
    if (N > 0) {
      rc = with_row<true>(dtype, V, [&](auto *form) {
        typedef typename std::remove_pointer<decltype(form)>::type Row;
        token_ratio_kernel<Row><<<row_blocks(N, Row::GL), group_threads(Row::GL), 0, st>>>(in, a);
        return launch_status("preference_score log-ratios");
      });
      if (rc != VK_OK) return rc;
    }
    if (B > 0 && B <= 64 && N <= PAIRS_AT_ONCE_TOKENS && P <= PAIRS_AT_ONCE_PAIRS) {
      pairs_at_once_kernel<<<1, 1024, 0, st>>>(token_ratio, lengths, pairs, static_cast<int>(P), static_cast<int>(B), T, beta,
                                               target, smoothing, inv_n, ratio, slope, margin, loss, coef);
    } else {
      if (B > 0) sequence_ratio_kernel<<<static_cast<unsigned>(B), 256, 0, st>>>(token_ratio, lengths, ratio, T);
      rc = launch_status("preference_score sequences");
      if (rc != VK_OK) return rc;
      pair_loss_kernel<<<1, 256, 0, st>>>(ratio, pairs, P, B, beta, target, smoothing, inv_n, margin, slope, loss);
      rc = launch_status("preference_score pairs");
      if (rc != VK_OK) return rc;
      if (B > 0)
        sequence_slope_kernel<<<static_cast<unsigned>((B + 3) / 4), 256, 0, st>>>(slope, pairs, lengths, P, B, coef);
    }
    rc = launch_status("preference_score slopes");
    if (rc != VK_OK) return rc;
  }
  if (!backward || N == 0) return VK_OK;
  return with_row<true>(dtype, V, [&](auto *form) {
    typedef typename std::remove_pointer<decltype(form)>::type Row;
    softmax_grad_kernel<Row><<<row_blocks(N, Row::GL), group_threads(Row::GL), 0, st>>>(in, a, coef, dlogits,
                                                                                       Upstream{upstream, unless_one});
    return launch_status("preference_score gradient");
  });
}

extern "C" int vk_distill_score(const void *logits, int32_t dtype, int64_t ld_b, int64_t ld_t, const void *values,
                                int32_t values_dtype, const void *ids, int32_t ids_64, int32_t K, const float *t_lse,
                                const float *weights, double temperature, int32_t mean, double inv_n, float *loss, float *kl,
                                void *dlogits, const float *upstream, int32_t unless_one, int64_t B, int64_t T, int32_t V,
                                void *ws, int64_t ws_bytes, void *stream) {
  int rc = check_rows("distill_score", logits, dtype, ld_b, ld_t, B, T, V);
  if (rc != VK_OK) return rc;
  VK_CHECK_ARG(K >= 1 && K <= LIST_MAX, "distill_score: lists of 1 to %d", LIST_MAX);
  VK_CHECK_ARG(values_dtype == VK_DTYPE_BF16 || values_dtype == VK_DTYPE_F32, "distill_score: list values are bf16 or fp32");
  VK_CHECK_ARG(temperature > 0.0 && temperature <= 1e30 && temperature >= 1e-30, "distill_score: the temperature must be positive");
  VK_CHECK_ARG(!unless_one || upstream, "distill_score: unless_one needs the upstream gradient");
  int64_t need;
  rc = vk_objective_workspace(B, T, 0, &need);
  if (rc != VK_OK) return rc;
  VK_CHECK_ARG(ws && vk_aligned16(ws) && ws_bytes >= need, "distill_score: the workspace needs %lld bytes", (long long)need);
  const int64_t N = B * T;
  VK_CHECK_ARG(N == 0 || (values && ids), "distill_score: null pointer");
  hipStream_t st = VK_STREAM(stream);
  double *weight_parts = static_cast<double *>(ws), *loss_parts = weight_parts + OBJ_PARTS;
  const Upstream up{upstream, unless_one};
  unsigned blocks = 0;
  if (N > 0) {
    const bool sums = mean && weights;
    const double scale = mean ? 1.0 / static_cast<double>(N) : inv_n;
    const LogitRows in{logits, ld_b, ld_t, N, static_cast<uint32_t>(T), V};
    DistillArgs a{values, values_dtype == VK_DTYPE_BF16, ids, ids_64, K, t_lse, weights, temperature,
                  1.0 / temperature, ExpScale::of(temperature), sums, scale, weight_parts, kl, dlogits,
                  loss ? loss_parts : nullptr, up};
    rc = with_row<false>(dtype, V, [&](auto *form) {
      typedef typename std::remove_pointer<decltype(form)>::type Row;
      if (sums && count_here(N, T, Row::GL, false))
        a.weight_parts = nullptr;
      else if (sums)
        weight_parts_kernel<<<OBJ_PARTS, 256, 0, st>>>(nullptr, nullptr, weights, weight_parts, N, V, up);
      const int rc2 = launch_status("distill_score weights");
      if (rc2 != VK_OK) return rc2;
      blocks = row_blocks(N, Row::GL);
      if constexpr (Row::GL == 16) {
        if (K <= 32) {
          distill_rows_kernel<Row, 32><<<blocks, group_threads(Row::GL), 0, st>>>(in, a);
          return launch_status("distill_score");
        }
      }
      distill_rows_kernel<Row, LIST_MAX><<<blocks, group_threads(Row::GL), 0, st>>>(in, a);
      return launch_status("distill_score");
    });
    if (rc != VK_OK) return rc;
  }
  if (!loss) return VK_OK;
  loss_join_kernel<<<1, 256, 0, st>>>(loss_parts, static_cast<int>(blocks), loss);
  return launch_status("distill_score loss");
}
