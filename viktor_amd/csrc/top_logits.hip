// The k largest logits of each row with their ids, in falling order (equal values: the lower id first), and the row's
// log-sum-exp: a teacher's list for distillation.
//
// The row stays in the registers of a wavefront (up to 512 logits, element lane + 64 i with lane `lane`; to 704 vectors of 16
// bytes, whole vectors) or of a workgroup. A bound that at least k logits reach comes from one or a few maxima a thread: bit
// by bit with ballots, the largest number that k of the maxima reach. What reaches it in the row (a little more than k logits
// of most rows) goes to shared memory with its id, and one wavefront sorts it in registers. Rows with more than 256 candidates
// have their k-th logit searched bit by bit over all of it, in memory, then the id up to which equal ones are taken: some 65
// walks. Those are rows of many equal logits, and any row just past 512 logits with a list that is long for it: a maximum of 16
// bytes bounds little where there are hardly more vectors than entries (bf16 rows of 513 to some 1250 logits with lists of nine
// tenths of their vectors or more, fp32 rows of 513 to 560 with lists of 120 or more). 16416 rows of 640 bf16: lists of 64 in 34
// us, of 100 in 254; of 1000: 39 for 100, 275 for 128; of 1200 and 1367: 319 and 107 for 128; of 520 fp32: 302 for 128; of 512
// bf16, whose bound is of single logits, 35 for 128.
// Rows of up to 32 logits go one a thread: each logit counts the ones before it.
// Logits of -inf and NaN are no entries: a list that runs out ends in id -1, value -inf.
//
// Bound by VALU issue: an exponential, two comparisons and two unpackings an element, and some 250 instructions a row for the
// bound and the sort. 2064 x 87383 bf16 at 3.6 TB/s of the 6.8 that reads reach, 16416 x 5463 bf16 at 3.1, 32896 x 343 at 0.9.
#include <float.h>

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

// A logit and its id as one number, larger ones first in the list: 64 bits, or 32 where the logit is a bf16 and the id
// fits 16.
template <typename Entry>
__device__ __forceinline__ Entry entry_of(float z, int id);
template <>
__device__ __forceinline__ uint64_t entry_of(float z, int id) {
  return (static_cast<uint64_t>(key_of(z)) << 32) | (0xffffffffu - static_cast<uint32_t>(id));
}
template <>
__device__ __forceinline__ uint32_t entry_of(float z, int id) {
  return (key_of(z) & 0xffff0000u) | (0xffffu - static_cast<uint32_t>(id));
}
__device__ __forceinline__ float value_of(uint64_t e) { return of_key(static_cast<uint32_t>(e >> 32)); }
__device__ __forceinline__ int id_of(uint64_t e) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(e)); }
// (a negative bf16's key has ones below)
__device__ __forceinline__ float value_of(uint32_t e) {
  return of_key(e & 0x80000000u ? e & 0xffff0000u : e | 0xffffu);
}
__device__ __forceinline__ int id_of(uint32_t e) { return static_cast<int>(0xffffu - (e & 0xffffu)); }

// Element lane + 64 i with lane `lane`: every lane has its share of a short row.
template <typename T, int NE>
struct RowStrided {
  typedef T type;
  static constexpr int GL = 64, TOP_WAVES = 8, TOP_MAXIMA = NE;
  float z[NE];

  template <int M>
  __device__ __forceinline__ void maxima(float (&m)[M]) const {
    static_assert(M == NE, "its elements");
#pragma unroll
    for (int i = 0; i < M; ++i) m[i] = z[i];
  }

  __device__ __forceinline__ void load(const T *p, int V, int lane) {
#pragma unroll
    for (int i = 0; i < NE; ++i) z[i] = lane + 64 * i < V ? load_one(p + lane + 64 * i) : -INFINITY;
  }
  __device__ __forceinline__ void keep() {}
  template <typename F>
  __device__ __forceinline__ void values(F f) const {
#pragma unroll
    for (int i = 0; i < NE; ++i) f(z[i]);
  }
  __device__ __forceinline__ float sum_near(float top, ExpScale scale) const {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NE; ++i) sum += exp_near(z[i], top, scale);
    return sum;
  }
  template <typename F>
  __device__ __forceinline__ void each(int lane, F f) const {
#pragma unroll
    for (int i = 0; i < NE; ++i) f(lane + 64 * i, z[i]);
  }
};

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

// A bound that k of a wavefront's keys reach, R keys a lane: the largest with zeros in its low half (BF16: the keys are of bf16
// values, which have nothing there) or in its low 12 bits, from its highest bit down; 0 where fewer than k keys are above 0.
template <int R, bool BF16>
__device__ __forceinline__ uint32_t kth_key(const uint32_t (&key)[R], int k) {
  uint32_t bound = 0;
#pragma unroll
  for (int bit = 31; bit >= (BF16 ? 16 : 12); --bit) {
    const uint32_t trial = bound | (1u << bit);
    int n = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) n += __popcll(__ballot(key[r] >= trial));
    if (n >= k) bound = trial;
  }
  return BF16 && bound && !(bound & 0x80000000u) ? bound | 0xffffu : bound;  // (a negative bf16's key has ones there)
}

// The lane's partner's word across j lanes (xor): data-parallel moves within rows of 16, one swizzle for 4, gfx950's lane swaps
// for 16 and 32. (ds_bpermute, which __shfl_xor is, goes through the LDS pipe with an address each time.)
template <int J>
__device__ __forceinline__ uint32_t across(uint32_t x) {
  if constexpr (J == 1) return __builtin_amdgcn_mov_dpp(x, 0xb1, 0xf, 0xf, true);        // quads 1 0 3 2
  if constexpr (J == 2) return __builtin_amdgcn_mov_dpp(x, 0x4e, 0xf, 0xf, true);        // quads 2 3 0 1
  if constexpr (J == 4) return __builtin_amdgcn_ds_swizzle(x, 0x101f);                   // lane ^ 4 of 32
  if constexpr (J == 8) return __builtin_amdgcn_mov_dpp(x, 0x128, 0xf, 0xf, true);       // rows of 16 turned by 8
  if constexpr (J == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return (threadIdx.x & 16) ? r[0] : r[1];
  }
  if constexpr (J == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return (threadIdx.x & 32) ? r[0] : r[1];
  }
  return x;
}
template <int J>
__device__ __forceinline__ uint64_t across(uint64_t x) {
  return (static_cast<uint64_t>(across<J>(static_cast<uint32_t>(x >> 32))) << 32) | across<J>(static_cast<uint32_t>(x));
}
template <typename Entry>
__device__ __forceinline__ Entry across(Entry x, int j) {  // (j is a constant where it is unrolled)
  switch (j) {
    case 1: return across<1>(x);
    case 2: return across<2>(x);
    case 4: return across<4>(x);
    case 8: return across<8>(x);
    case 16: return across<16>(x);
    default: return across<32>(x);
  }
}

// Sorts 64 R entries of a wavefront, entry 64 r + lane with e[r], the largest first (bitonic).
template <typename Entry, int R>
__device__ __forceinline__ void sort_entries(Entry (&e)[R], int lane) {
#pragma unroll
  for (int k = 2; k <= 64 * R; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j >= 64) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int q = r ^ (j >> 6);
          if (q > r) {
            const bool falls = ((64 * r + lane) & k) == 0 || k == 64 * R;
            const Entry hi = e[r] > e[q] ? e[r] : e[q], lo = e[r] > e[q] ? e[q] : e[r];
            e[r] = falls ? hi : lo;
            e[q] = falls ? lo : hi;
          }
        }
      } else {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const bool falls = ((64 * r + lane) & k) == 0 || k == 64 * R, first = (lane & j) == 0;
          const Entry o = across(e[r], j);
          e[r] = (falls == first) == (e[r] > o) ? e[r] : o;
        }
      }
    }
  }
}

// What a row's log-sum-exp has beyond its maximum, from the sum of exponentials by it (by 0 where it is infinite: NaN then if
// a logit is).
__device__ __forceinline__ double log_beyond(float top, float s) { return isinf(top) && !isnan(s) ? 0.0 : log_near(s); }

template <typename T>
__device__ __forceinline__ void write_entry(T *values, int32_t *ids, int64_t at, float value, int id) {
  store_one(values + at, value);
  ids[at] = id;
}

// Entries entry(0), ... of a wavefront, 64 R at most (0 where there is none), sorted; the first K written.
template <typename T, typename Entry, int R, typename F>
__device__ __forceinline__ void sort_and_write(F entry, int K, T *values, int32_t *ids, int64_t at, int lane) {
  Entry e[R];
#pragma unroll
  for (int r = 0; r < R; ++r) e[r] = entry(64 * r + lane);
  sort_entries<Entry, R>(e, lane);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int place = 64 * r + lane;
    if (place < K) write_entry(values, ids, at + place, e[r] ? value_of(e[r]) : -INFINITY, e[r] ? id_of(e[r]) : -1);
  }
  for (int place = 64 * R + lane; place < K; place += 64) write_entry(values, ids, at + place, -INFINITY, -1);
}

template <typename Row, typename Entry>
__global__ __launch_bounds__(group_threads(Row::GL), Row::TOP_WAVES) void top_rows_kernel(
    const void *logits, int64_t ld_b, int64_t ld_t, int64_t N, uint32_t T_, int V, int K, ExpScale scale, double inv_tau,
    void *values_, int32_t *ids, float *lse) {
  typedef typename Row::type T;
  constexpr int GL = Row::GL, GROUPS = group_threads(GL) / GL, WAVES = GL / 64;
  // candidates of a wavefront
  constexpr int OWN = WAVES == 1 ? 512 : WAVES <= 4 ? 256 : 128;
  __shared__ Entry cand[GROUPS * WAVES][OWN];
  __shared__ int found[GROUPS * WAVES], taken[GROUPS];
  __shared__ float sh[WAVES];
  __shared__ decltype(Row().sum_near(0.f, ExpScale())) sums[WAVES];
  __shared__ int shc[WAVES];
  __shared__ uint32_t maxima[GL > 64 ? GL : 1], bound_sh;
  const int lane = lane_of<GL>(), group = group_of<GL>(), l64 = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Entry *own = cand[wave];
  T *values = static_cast<T *>(values_);
  int turn = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * GROUPS + group; row < N;
       row += static_cast<int64_t>(gridDim.x) * GROUPS) {
    const uint32_t b = static_cast<uint32_t>(row) / T_, t = static_cast<uint32_t>(row) % T_;
    const T *z = static_cast<const T *>(logits) + b * ld_b + t * ld_t;
    Row r;
    r.load(z, V, lane);
    float mine = -INFINITY;
    r.values([&](float x) { mine = fmaxf(mine, x); });
    r.keep();
    // A bound from the threads' maxima: by the wavefront itself or, in a workgroup, by one of its wavefronts in turn while the
    // others are at their sums.
    float top;
    uint32_t bound = 0;
    if constexpr (GL == 64) {
      top = group_max<GL>(mine, sh);
      // from one maximum a lane for short lists, from several for longer ones (a bound from M maxima leaves some
      // -M log(1 - K / M) candidates)
      if (K <= 32) {
        const uint32_t key[1] = {key_of(mine)};
        bound = kth_key<1, sizeof(T) == 2>(key, K);
      } else {
        constexpr int M = Row::TOP_MAXIMA;
        float m[M];
        r.maxima(m);
        r.keep();
        uint32_t key[M];
#pragma unroll
        for (int i = 0; i < M; ++i) key[i] = key_of(m[i]);
        bound = kth_key<M, sizeof(T) == 2>(key, K);
      }
    } else {
      maxima[threadIdx.x] = key_of(mine);
      top = group_max<GL>(mine, sh);  // (a barrier for the maxima too)
      if (wave == turn) {
        uint32_t key[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) key[w] = maxima[64 * w + l64];
        const uint32_t k = kth_key<WAVES, sizeof(T) == 2>(key, K);
        if (l64 == 0) bound_sh = k;
      }
      turn = (turn + 1) % WAVES;
    }
    const auto part = r.sum_near(isinf(top) ? 0.f : top, scale);
    r.keep();
    const float s = static_cast<float>(group_add<GL>(part, sums));
    if constexpr (GL > 64) bound = bound_sh;
    if (lane == 0)
      lse[row] = static_cast<float>(static_cast<double>(top) * inv_tau + log_beyond(top, s));
    // each wavefront's candidates, in its own part of the list
    const float least = bound ? of_key(bound) : -FLT_MAX;
    int n = 0;
    r.each(lane, [&](int i, float x) {
      const uint64_t m = __ballot(x >= least);
      if (m) {
        const int at = n + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(m >> 32),
                                                     __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(m), 0));
        if (x >= least && at < OWN) own[at] = entry_of<Entry>(x, i);
        n += __popcll(m);
      }
    });
    int C = n;
    bool fits = n <= OWN;
    if constexpr (GL > 64) {
      if (l64 == 0) found[wave] = n;
      __syncthreads();
      C = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const int f = found[w];
        fits &= f <= OWN;
        C += f;
      }
    }
    const int64_t at = row * K;
    if (fits && C <= 256) {
      group_sync<64>();
      if (lane < 64) {
        // entry e of all wavefronts' parts together
        auto entry = [&](int e) -> Entry {
          if (WAVES == 1) return e < C ? own[e] : 0;
          int w = 0;
#pragma unroll
          for (int k = 0; k < WAVES - 1; ++k) {
            const int f = found[k];
            if (w == k && e >= f) {
              e -= f;
              w = k + 1;
            }
          }
          return e < found[w] ? cand[w][e] : 0;
        };
        if (C <= 64)
          sort_and_write<T, Entry, 1>(entry, K, values, ids, at, lane);
        else if (C <= 128)
          sort_and_write<T, Entry, 2>(entry, K, values, ids, at, lane);
        else
          sort_and_write<T, Entry, 4>(entry, K, values, ids, at, lane);
      }
    } else {
      // the k-th key, bit by bit over the row (more candidates than K, all above -inf), then the ids of its equals. (Walked in
      // memory: the registers of a form for this would be every row's.)
      RowWalk<T, GL> w;
      w.load(z, V, lane);
      uint32_t kth = 0;
      for (int bit = 31; bit >= 0; --bit) {
        const uint32_t trial = kth | (1u << bit);
        const float f = of_key(trial);
        int c = 0;
        w.values([&](float x) { c += x >= f ? 1 : 0; });
        if (group_count<GL>(c, shc) >= K) kth = trial;
      }
      const float f = of_key(kth);
      int c = 0;
      w.values([&](float x) { c += x > f ? 1 : 0; });
      const int want = K - group_count<GL>(c, shc);
      uint32_t last = 0;  // the largest id bound that has fewer than `want` equals below it
      for (int bit = 30; bit >= 0; --bit) {
        const uint32_t trial = last | (1u << bit);
        c = 0;
        w.each(lane, [&](int i, float x) { c += (x == f && static_cast<uint32_t>(i) < trial) ? 1 : 0; });
        if (group_count<GL>(c, shc) < want) last = trial;
      }
      if (lane == 0) taken[group] = 0;
      group_sync<GL>();
      Entry *first = cand[group * WAVES];  // (K <= 128 <= OWN)
      w.each(lane, [&](int i, float x) {
        if (x > f || (x == f && static_cast<uint32_t>(i) <= last)) first[atomicAdd(&taken[group], 1)] = entry_of<Entry>(x, i);
      });
      group_sync<GL>();
      if (lane < 64) {
        auto entry = [&](int e) -> Entry { return e < K ? first[e] : 0; };
        sort_and_write<T, Entry, 2>(entry, K, values, ids, at, lane);
      }
    }
    group_sync<GL>();
  }
}

// Rows of up to NE logits, one a thread.
template <typename T, int NE>
__global__ __launch_bounds__(256) void top_lanes_kernel(const void *logits, int64_t ld_b, int64_t ld_t, int64_t N, uint32_t T_,
                                                       int V, int K, ExpScale scale, double inv_tau, void *values,
                                                       int32_t *ids, float *lse) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (row >= N) return;
  const uint32_t b = static_cast<uint32_t>(row) / T_, t = static_cast<uint32_t>(row) % T_;
  RowLane<T, NE> r;
  r.load(static_cast<const T *>(logits) + b * ld_b + t * ld_t, V, 0);
  float top = -INFINITY, s = 0.f;
  r.values([&](float x) { top = fmaxf(top, x); });
  const float base = isinf(top) ? 0.f : top;
  r.values([&](float x) { s += exp_of(x, base, scale); });
  lse[row] = static_cast<float>(static_cast<double>(top) * inv_tau + log_beyond(top, s));
  uint32_t key[NE];
  int entries = 0;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    key[i] = key_of(r.z[i]);
    entries += key[i] ? 1 : 0;
  }
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    int place = 0;
#pragma unroll
    for (int j = 0; j < NE; ++j) place += (j < i ? key[j] >= key[i] : key[j] > key[i]) ? 1 : 0;
    if (key[i] && place < K) write_entry(static_cast<T *>(values), ids, row * K + place, of_key(key[i]), i);
  }
  for (int place = entries; place < K; ++place) write_entry(static_cast<T *>(values), ids, row * K + place, -INFINITY, -1);
}

// row_form for rows of more than 512 logits, with 512 threads where 1024 would do: two workgroups a CU, of which one loads
// while the other sorts (2064 x 87383 bf16, lists of 64: 100 us; 1024 threads 199). A
// wavefront a row to 704 vectors: 16416 x 5463 bf16, lists of 8 and 64, 50 and 72 us, 91 and 114 with 256 threads.
template <typename F>
int top_form(int64_t vectors, F f) {
#define VK_FORM(GL, NV) \
  if (vectors <= GL * NV) return f(std::integral_constant<int, GL>{}, std::integral_constant<int, NV>{})
  VK_FORM(64, 3);
  VK_FORM(64, 6);
  VK_FORM(64, 11);
  VK_FORM(256, 6);
  VK_FORM(256, 11);
  VK_FORM(512, 11);
  VK_FORM(512, 22);
  VK_FORM(1024, 22);
#undef VK_FORM
  return f(std::integral_constant<int, 1024>{}, std::integral_constant<int, 0>{});
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
  auto run = [&](auto kernel, int threads, int groups, bool all) {
    const int64_t want = (N + groups - 1) / groups, most = static_cast<int64_t>(device_cus_cached()) * (2048 / threads);
    kernel<<<static_cast<unsigned>(all || want < most ? want : most), threads, 0, VK_STREAM(stream)>>>(
        logits, ld_b, ld_t, N, static_cast<uint32_t>(T), V, K, scale, 1.0 / temperature, values, ids, lse);
    return launch_status("top_logits");
  };
  auto launch = [&](auto elem) {
    typedef decltype(elem) E;
    typedef typename std::conditional<sizeof(E) == 2, uint32_t, uint64_t>::type Short;
    if (V <= 8) return run(top_lanes_kernel<E, 8>, 256, 256, true);
    if (V <= 16) return run(top_lanes_kernel<E, 16>, 256, 256, true);
    if (V <= 32) return run(top_lanes_kernel<E, 32>, 256, 256, true);
    if (V <= 256) return run(top_rows_kernel<RowStrided<E, 4>, Short>, 256, 4, false);
    if (V <= 384) return run(top_rows_kernel<RowStrided<E, 6>, Short>, 256, 4, false);
    if (V <= 512) return run(top_rows_kernel<RowStrided<E, 8>, Short>, 256, 4, false);
    return top_form((V + kVec<E> - 1) / kVec<E>, [&](auto gl, auto nv) {
      constexpr int G = decltype(gl)::value;
      typedef typename RowForm<E, G, decltype(nv)::value>::type Row;
      if (V <= 65536) return run(top_rows_kernel<Row, Short>, group_threads(G), group_threads(G) / G, false);
      return run(top_rows_kernel<Row, uint64_t>, group_threads(G), group_threads(G) / G, false);
    });
  };
  return dtype == VK_DTYPE_BF16 ? launch(bf16_t{}) : launch(float{});
}
