// The k largest logits of each row with their ids, in falling order (equal values: the lower id first), and the row's
// log-sum-exp: a teacher's list for distillation.
//
// The row stays in registers. A bound that at least k logits reach comes from one value a thread: each wavefront finds the
// ceil(k / wavefronts)-th largest of its lanes' maxima, bit by bit with ballots, and the least of these bounds the row's
// k-th logit from below. What reaches it (a little more than k logits of most rows) goes to shared memory, where each
// candidate counts the ones before it: its place in the list. Rows with more candidates than fit (many equal logits, lists
// nearly as long as the row) have their k-th logit searched bit by bit over all of it, then the id up to which equal ones
// are taken. Logits of -inf and NaN are no entries: a list that runs out ends in id -1, value -inf.
#include "common.h"
#include "vocab_rows.h"

namespace vk {

constexpr int TOP_MAX = 128;

// Order-preserving keys of floats above -inf: larger logits have larger keys, both zeros the same; 0 for -inf and NaN.
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t u = __float_as_uint(z + 0.f);
  const uint32_t k = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
  return z > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// Sum of an int over the group; callable again at once.
template <int GL>
__device__ __forceinline__ int group_count(int v, int *sh) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  if constexpr (GL > 64) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < GL / 64; ++w) v += sh[w];
    __syncthreads();
  }
  return v;
}

template <typename Row>
__global__ __launch_bounds__(group_threads(Row::GL)) void top_rows_kernel(const void *logits, int64_t ld_b, int64_t ld_t,
                                                                         int64_t N, uint32_t T_, int V, int K, ExpScale scale,
                                                                         double inv_tau, void *values, int32_t *ids,
                                                                         float *lse) {
  typedef typename Row::type T;
  constexpr int GL = Row::GL, GROUPS = group_threads(GL) / GL, WAVES = GL / 64;
  constexpr int CAP = GL == 64 ? 256 : 512;  // candidates
  __shared__ uint64_t cand[GROUPS][CAP];
  __shared__ int taken[GROUPS];
  __shared__ float sh[2][WAVES];
  __shared__ int shc[WAVES];
  __shared__ uint32_t shk[WAVES];
  const int lane = threadIdx.x % GL, group = threadIdx.x / GL;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group; row < N;
       row += static_cast<int64_t>(gridDim.x) * GROUPS) {
    const uint32_t b = static_cast<uint32_t>(row) / T_, t = static_cast<uint32_t>(row) % T_;
    const T *z = static_cast<const T *>(logits) + b * ld_b + t * ld_t;
    Row r;
    r.load(z, V, lane);
    if (lane == 0) taken[group] = 0;
    float mine = -INFINITY;
    r.values([&](float x) { mine = fmaxf(mine, x); });
    const float top = group_max<GL>(mine, sh[0]);
    // the wavefront's bound
    const int share = (K + WAVES - 1) / WAVES;
    uint32_t bound = 0;
    if (share <= 64) {
      const uint32_t key = key_of(mine);
      constexpr int LOW = sizeof(T) == 2 ? 16 : 0;  // (a bf16's low bits say nothing)
#pragma unroll
      for (int bit = 31; bit >= LOW; --bit) {
        const uint32_t trial = bound | (1u << bit);
        if (__popcll(__ballot(key >= trial)) >= share) bound = trial;
      }
      // (a negative bf16's key has ones there)
      if (LOW && bound && !(bound & 0x80000000u)) bound |= 0xffffu;
    }
    if constexpr (GL > 64) {
      if ((threadIdx.x & 63) == 0) shk[threadIdx.x >> 6] = bound;
    }
    float s = 0.f;
    r.values([&](float x) { s += exp_of(x, top, scale); });
    s = group_add<GL>(s, sh[1]);
    if constexpr (GL > 64) {
      bound = shk[0];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) bound = min(bound, shk[w]);
    }
    group_sync<GL>();
    if (lane == 0) lse[row] = static_cast<float>(static_cast<double>(top) * inv_tau + (top == -INFINITY ? 0.0 : log_of(s)));
    // candidates
    const float floor = bound ? of_key(bound) : -INFINITY;
    int n = 0;
    r.values([&](float x) { n += (x >= floor && x > -INFINITY) ? 1 : 0; });
    int at = n ? atomicAdd(&taken[group], n) : 0;
    group_sync<GL>();
    int C = taken[group];
    group_sync<GL>();
    if (C <= CAP) {
      if (n)
        r.each(lane, [&](int i, float x) {
          if (x >= floor && x > -INFINITY) cand[group][at++] = (static_cast<uint64_t>(key_of(x)) << 32) | (0xffffffffu - i);
        });
    } else {
      // the k-th key, bit by bit over the row (more than CAP >= K logits are above -inf), then the ids of its equals
      uint32_t kth = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t trial = kth | (1u << bit);
        const float f = of_key(trial);
        int c = 0;
        r.values([&](float x) { c += x >= f ? 1 : 0; });
        if (group_count<GL>(c, shc) >= K) kth = trial;
      }
      const float f = of_key(kth);
      int c = 0;
      r.values([&](float x) { c += x > f ? 1 : 0; });
      const int want = K - group_count<GL>(c, shc);
      uint32_t last = 0;  // the largest id bound that has fewer than `want` equals below it
      for (int bit = 30; bit >= 0; --bit) {
        const uint32_t trial = last | (1u << bit);
        c = 0;
        r.each(lane, [&](int i, float x) { c += (x == f && static_cast<uint32_t>(i) < trial) ? 1 : 0; });
        if (group_count<GL>(c, shc) < want) last = trial;
      }
      if (lane == 0) taken[group] = 0;
      group_sync<GL>();
      r.each(lane, [&](int i, float x) {
        if (x > f || (x == f && static_cast<uint32_t>(i) <= last))
          cand[group][atomicAdd(&taken[group], 1)] = (static_cast<uint64_t>(key_of(x)) << 32) | (0xffffffffu - i);
      });
      C = K;
    }
    group_sync<GL>();
    // each candidate's place
    for (int i = lane; i < C; i += GL) {
      const uint64_t me = cand[group][i];
      int place = 0;
      for (int j = 0; j < C; ++j) place += cand[group][j] > me ? 1 : 0;
      if (place < K) {
        store_one(static_cast<T *>(values) + row * K + place, of_key(static_cast<uint32_t>(me >> 32)));
        ids[row * K + place] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(me));
      }
    }
    for (int i = C + lane; i < K; i += GL) {
      store_one(static_cast<T *>(values) + row * K + i, -INFINITY);
      ids[row * K + i] = -1;
    }
    group_sync<GL>();
  }
}

}  // namespace vk

using namespace vk;

extern "C" int vk_top_logits(const void *logits, int32_t dtype, int64_t ld_b, int64_t ld_t, int32_t K, double temperature,
                             void *values, int32_t *ids, float *lse, int64_t B, int64_t T, int32_t V, void *stream) {
  VK_CHECK_ARG(dtype == VK_DTYPE_BF16 || dtype == VK_DTYPE_F32, "top_logits: logits are bf16 or fp32");
  VK_CHECK_ARG(B >= 0 && T >= 0 && V > 0 && V <= (1 << 30) && B < (int64_t(1) << 31) && T < (int64_t(1) << 31) &&
                   B * T < (int64_t(1) << 31),
               "top_logits: bad sizes");
  VK_CHECK_ARG(K >= 1 && K <= TOP_MAX && K <= V, "top_logits: lists of 1 to %d, no longer than the row", TOP_MAX);
  VK_CHECK_ARG(temperature > 0.0 && temperature <= 1e30 && temperature >= 1e-30, "top_logits: the temperature must be positive");
  const int64_t N = B * T;
  if (N == 0) return VK_OK;
  VK_CHECK_ARG(logits && values && ids && lse, "top_logits: null pointer");
  VK_CHECK_ARG((T < 2 || ld_t >= V) && (B < 2 || ld_b >= V) && ld_t >= 0 && ld_b >= 0, "top_logits: rows overlap");
  const ExpScale scale = ExpScale::of(temperature);
  auto launch = [&](auto elem) {
    typedef decltype(elem) E;
    return row_form((V + kVec<E> - 1) / kVec<E>, [&](auto gl, auto nv) {
      constexpr int G = decltype(gl)::value < 64 ? 64 : decltype(gl)::value;
      constexpr int NV = decltype(gl)::value < 64 ? 2 : decltype(nv)::value;  // 16 lanes of 3 or 6 vectors: 64 of 2
      typedef typename RowForm<E, G, NV>::type Row;
      constexpr int threads = group_threads(G), groups = threads / G;
      const int64_t want = (N + groups - 1) / groups, most = static_cast<int64_t>(device_cus_cached()) * (2048 / threads);
      top_rows_kernel<Row><<<static_cast<unsigned>(want < most ? want : most), threads, 0, VK_STREAM(stream)>>>(
          logits, ld_b, ld_t, N, static_cast<uint32_t>(T), V, K, scale, 1.0 / temperature, values, ids, lse);
      return launch_status("top_logits");
    });
  };
  return dtype == VK_DTYPE_BF16 ? launch(bf16_t{}) : launch(float{});
}
