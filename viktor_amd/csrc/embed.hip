// The token embedding at vocabularies past the 4-mers': the lookup of scaled rows and the table's gradient.
//
// Lookup: out[r, :] = round(scale * W[t_r, :]), the product in fp32. Ids outside [0, V) give zero rows.
//
// Gradient: g[v, :] = scale * sum over t_r = v of dY[r, :], fp32, without atomics on floats. Rows are brought into token
// order first (a stable sort of the ids, row numbers as its payload), so that every vocabulary row is one run of
// consecutive sorted positions in ascending row order; its sum then reads each gradient row once, in an order that only
// n, V and the ids decide. Ids outside [0, V), and `pad`, get the key V: they sort behind every row and no sum reads
// them. The sort:
//   n <= ES_RANK_MAX: the position of a row is a count, pos = #{key_j < key_i} + #{j < i: key_j = key_i}, taken over all
//     n keys in LDS; the same loop gives the run's length, so one launch sorts and finds the runs;
//   larger n: radix passes over digits of at most 9 bits (2 for the vocabularies of k = 6 .. 8), each a histogram per
//     tile, a scan per digit over the tiles, and a stable scatter.
// A run of up to ES_CHUNK rows is summed by one group of lanes. A longer one is cut at multiples of ES_CHUNK sorted
// positions, so that a token that most rows share (padding, a homopolymer) spreads over the chip: each chunk writes the
// partial sum of its first run and of its last run (no more than these two can be longer than a chunk), and the join
// adds a run's partials in chunk order.
#include "row_access.h"

namespace vk {

constexpr int EL_ROWS = 4;  // rows whose loads a lane has in flight

// LPR lanes share a row (64 / LPR rows per wavefront side by side), N elements each: 16-byte accesses of the narrower
// type where both are bf16, of the fp32 side otherwise.
template <typename WT, typename OT, int LPR>
__global__ __launch_bounds__(256) void embed_lookup_kernel(const WT *__restrict__ w, const int64_t *__restrict__ tokens,
                                                           int64_t n, int64_t V, int d, float scale,
                                                           OT *__restrict__ out) {
  constexpr int N = sizeof(WT) + sizeof(OT) == 4 ? 8 : 4;
  const int lane = threadIdx.x & 63, sub = lane / LPR, c0 = (lane % LPR) * N;
  constexpr int SIDE = 64 / LPR;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t r0 = wave * (EL_ROWS * SIDE) + sub;
  int64_t t[EL_ROWS];
#pragma unroll
  for (int u = 0; u < EL_ROWS; ++u) t[u] = r0 + u * SIDE < n ? tokens[r0 + u * SIDE] : -1;
  for (int c = c0; c < d; c += LPR * N) {
    const bool whole = c + N <= d;
    float v[EL_ROWS][N];
#pragma unroll
    for (int u = 0; u < EL_ROWS; ++u) {
      const bool in = t[u] >= 0 && t[u] < V;
      const WT *src = w + (in ? t[u] : 0) * d + c;
      if (whole) {
        load_row<N>(src, v[u]);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[u][k] = c + k < d ? load_one(src + k) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < N; ++k) v[u][k] = in ? v[u][k] * scale : 0.f;
    }
#pragma unroll
    for (int u = 0; u < EL_ROWS; ++u) {
      const int64_t r = r0 + u * SIDE;
      if (r >= n) continue;
      OT *dst = out + r * d + c;
      if (whole) {
        store_row<N>(dst, v[u]);
      } else {
        for (int k = 0; k < N && c + k < d; ++k) store_one(dst + k, v[u][k]);
      }
    }
  }
}

// ---- the sort ----------------------------------------------------------------------------------------------------------

constexpr int ES_RANK_MAX = 4096;  // rows that the counting sort takes
constexpr int ES_RANK_ROWS = 16;   // rows per workgroup of it
constexpr int ES_TILE = 2048;      // keys per workgroup of a radix pass: 8 per thread
constexpr int ES_BITS = 9;         // digit bits at most
constexpr int ES_CHUNK = 64;       // sorted positions per chunk

struct Run {
  int32_t start, end;
};

__device__ __forceinline__ uint32_t sort_key(int64_t t, int32_t V, int64_t pad) {
  return t >= 0 && t < V && t != pad ? static_cast<uint32_t>(t) : static_cast<uint32_t>(V);
}

__global__ __launch_bounds__(256) void embed_runs_clear_kernel(Run *__restrict__ runs, int32_t V) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < V) runs[i] = Run{0, 0};
}

// 16 rows per workgroup, 16 threads each over a sixteenth of the keys.
__global__ __launch_bounds__(256) void embed_rank_kernel(const int64_t *__restrict__ tokens, int32_t n, int32_t V,
                                                         int64_t pad, uint32_t *__restrict__ keys,
                                                         int32_t *__restrict__ rows, Run *__restrict__ runs) {
  __shared__ uint32_t key[ES_RANK_MAX];
  for (int j = threadIdx.x; j < n; j += 256) key[j] = sort_key(tokens[j], V, pad);
  __syncthreads();
  const int part = threadIdx.x & 15;
  const int i = blockIdx.x * ES_RANK_ROWS + (threadIdx.x >> 4);
  const bool live = i < n;
  const uint32_t mine = key[live ? i : 0];
  int less = 0, same = 0, before = 0;
  for (int j = part; j < n; j += 16) {
    const uint32_t k = key[j];
    less += k < mine;
    same += k == mine;
    before += k == mine && j < i;
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    less += __shfl_xor(less, o, 64);
    same += __shfl_xor(same, o, 64);
    before += __shfl_xor(before, o, 64);
  }
  if (live && part == 0) {
    keys[less + before] = mine;
    rows[less + before] = i;
    if (before == 0 && mine < static_cast<uint32_t>(V)) runs[mine] = Run{less, less + same};
  }
}

// counts [bins, tiles]: keys of each digit in each tile. The first pass takes the ids themselves and clears the runs.
template <bool FIRST>
__global__ __launch_bounds__(256) void embed_hist_kernel(const int64_t *__restrict__ tokens,
                                                         const uint32_t *__restrict__ keys, int64_t n, int32_t V,
                                                         int64_t pad, int shift, int bins, uint32_t *__restrict__ counts,
                                                         Run *__restrict__ runs) {
  __shared__ uint32_t h[1 << ES_BITS];
  for (int b = threadIdx.x; b < bins; b += 256) h[b] = 0;
  if (FIRST)
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < V; i += static_cast<int64_t>(gridDim.x) * 256)
      runs[i] = Run{0, 0};
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * ES_TILE;
#pragma unroll
  for (int u = 0; u < ES_TILE / 256; ++u) {
    const int64_t i = base + u * 256 + threadIdx.x;
    if (i < n) {
      const uint32_t k = FIRST ? sort_key(tokens[i], V, pad) : keys[i];
      atomicAdd(&h[(k >> shift) & (bins - 1)], 1u);
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += 256) counts[static_cast<int64_t>(b) * gridDim.x + blockIdx.x] = h[b];
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t up = __shfl_up(v, o, 64);
    if (lane >= o) v += up;
  }
  return v;
}

// One wavefront per digit: counts[b, :] becomes its exclusive prefix over the tiles, totals[b] its sum.
__global__ __launch_bounds__(64) void embed_scan_kernel(uint32_t *__restrict__ counts, int tiles,
                                                        uint32_t *__restrict__ totals) {
  uint32_t *row = counts + static_cast<int64_t>(blockIdx.x) * tiles;
  const int lane = threadIdx.x;
  uint32_t run = 0;
  for (int t0 = 0; t0 < tiles; t0 += 64) {
    const uint32_t v = t0 + lane < tiles ? row[t0 + lane] : 0;
    const uint32_t inc = wave_scan(v, lane);
    if (t0 + lane < tiles) row[t0 + lane] = run + inc - v;
    run += __shfl(inc, 63, 64);
  }
  if (lane == 0) totals[blockIdx.x] = run;
}

// A stable scatter: wavefront w of a tile owns its keys 512 w .. 512 w + 511 in 8 rounds of 64, so (w, round, lane) is
// the keys' order. In a round the lanes of one digit find each other by a ballot per digit bit; a key's rank is the
// digit's count in this wavefront's earlier rounds plus its lanes below.
template <bool FIRST>
__global__ __launch_bounds__(256) void embed_scatter_kernel(const int64_t *__restrict__ tokens,
                                                            const uint32_t *__restrict__ keys_in,
                                                            const int32_t *__restrict__ rows_in, int64_t n, int32_t V,
                                                            int64_t pad, int shift, int bits,
                                                            const uint32_t *__restrict__ counts,
                                                            const uint32_t *__restrict__ totals,
                                                            uint32_t *__restrict__ keys_out,
                                                            int32_t *__restrict__ rows_out) {
  constexpr int BINS = 1 << ES_BITS, ROUNDS = ES_TILE / 256;
  __shared__ uint32_t wcount[4][BINS];
  __shared__ uint32_t wsum[4];
  const int bins = 1 << bits;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  for (int b = tid; b < 4 * BINS; b += 256) (&wcount[0][0])[b] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * ES_TILE + wid * (ES_TILE / 4);
  uint32_t key[ROUNDS];
  int32_t row[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int64_t i = base + r * 64 + lane;
    const bool in = i < n;
    key[r] = in ? (FIRST ? sort_key(tokens[i], V, pad) : keys_in[i]) : 0;
    row[r] = FIRST ? static_cast<int32_t>(i) : (in ? rows_in[i] : 0);
  }
  volatile uint32_t *mine = wcount[wid];
  const uint64_t below_mask = (uint64_t(1) << lane) - 1;
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const bool in = base + r * 64 + lane < n;
    const uint32_t dig = (key[r] >> shift) & (bins - 1);
    uint64_t peers = __ballot(in);
    for (int b = 0; b < bits; ++b) {
      const bool bit = (dig >> b) & 1;
      const uint64_t m = __ballot(bit);
      peers &= bit ? m : ~m;
    }
    const int below = __popcll(peers & below_mask);
    const uint32_t old = mine[dig];  // every lane reads before a digit's first lane writes (one wavefront, in order)
    rank[r] = static_cast<int32_t>(old) + below;
    if (in && below == 0) mine[dig] = old + static_cast<uint32_t>(__popcll(peers));
  }
  __syncthreads();
  // wcount[w][b]: first position of wavefront w's keys of digit b = keys of smaller digits + of this digit in earlier
  // tiles + in this tile's earlier wavefronts. Thread t scans digits 2 t and 2 t + 1
  const uint32_t t0 = 2 * tid < bins ? totals[2 * tid] : 0, t1 = 2 * tid + 1 < bins ? totals[2 * tid + 1] : 0;
  const uint32_t inc = wave_scan(t0 + t1, lane);
  if (lane == 63) wsum[wid] = inc;
  __syncthreads();
  uint32_t first = inc - t0 - t1;
  for (int w = 0; w < wid; ++w) first += wsum[w];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int b = 2 * tid + q;
    if (b < bins) {
      uint32_t at = first + (q ? t0 : 0) + counts[static_cast<int64_t>(b) * gridDim.x + blockIdx.x];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t c = wcount[w][b];
        wcount[w][b] = at;
        at += c;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (base + r * 64 + lane < n) {
      const uint32_t at = wcount[wid][(key[r] >> shift) & (bins - 1)] + rank[r];
      keys_out[at] = key[r];
      rows_out[at] = row[r];
    }
}

__global__ __launch_bounds__(256) void embed_runs_kernel(const uint32_t *__restrict__ keys, int64_t n, int32_t V,
                                                         Run *__restrict__ runs) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n) return;
  const uint32_t k = keys[i];
  if (k >= static_cast<uint32_t>(V)) return;
  if (i == 0 || keys[i - 1] != k) runs[k].start = static_cast<int32_t>(i);
  if (i == n - 1 || keys[i + 1] != k) runs[k].end = static_cast<int32_t>(i + 1);
}

// ---- the sums ----------------------------------------------------------------------------------------------------------

// Sum over sorted positions [p0, p1) of the gradient rows, for this lane's NCH groups of 4 columns (c, c + 4 LPR, ...):
// SIDE = 64 / LPR groups of lanes take every SIDE-th position and are added in a fixed order at the end, so every lane of
// a column has the sum. U positions' loads are in flight together.
template <typename T, int LPR, int NCH>
__device__ __forceinline__ void sum_rows(const T *__restrict__ drows, int64_t ld, const int32_t *__restrict__ rows,
                                         int p0, int p1, int c, int cols, float (&acc)[NCH][4]) {
  constexpr int SIDE = 64 / LPR, U = 8 / NCH < 2 ? 2 : 8 / NCH;
  const int sub = (threadIdx.x & 63) / LPR;
#pragma unroll
  for (int q = 0; q < NCH; ++q)
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[q][k] = 0.f;
  for (int p = p0 + sub; p < p1; p += U * SIDE) {
    float v[U][NCH][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int pu = p + u * SIDE;
      const bool in = pu < p1;
      const T *src = drows + static_cast<int64_t>(rows[in ? pu : p]) * ld + c;
#pragma unroll
      for (int q = 0; q < NCH; ++q) {
        const int cq = c + q * 4 * LPR;
        if (in && cq + 4 <= cols) {
          load_row<4>(src + q * 4 * LPR, v[u][q]);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) v[u][q][k] = in && cq + k < cols ? load_one(src + q * 4 * LPR + k) : 0.f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < NCH; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[q][k] += v[u][q][k];
  }
#pragma unroll
  for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
    for (int q = 0; q < NCH; ++q)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[q][k] += __shfl_xor(acc[q][k], o, 64);
}

__device__ __forceinline__ void put4(float *dst, int c, int cols, const float (&v)[4], float scale, bool add) {
  if (c + 4 <= cols) {
    f32x4_e o = {v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale};
    if (add) o += *reinterpret_cast<const f32x4_e *>(dst);
    *reinterpret_cast<f32x4_e *>(dst) = o;
  } else {
    for (int k = 0; k < 4 && c + k < cols; ++k) dst[k] = add ? dst[k] + v[k] * scale : v[k] * scale;
  }
}

// Wavefronts 0 .. chunks - 1: one chunk's partial sums of the long runs in it (slot 0: the run at its first position,
// slot 1: the run at its last, where that is another one). The others: one vocabulary row each, unless its run is long;
// a row without a run is zero (accumulate: left as it is). grid.y: blocks of 4 LPR NCH columns.
template <typename T, int LPR, int NCH>
__global__ __launch_bounds__(256) void embed_sum_kernel(const T *__restrict__ drows, int64_t ld, int32_t n, int32_t V,
                                                        int d, const uint32_t *__restrict__ keys,
                                                        const int32_t *__restrict__ rows, const Run *__restrict__ runs,
                                                        int32_t chunks, float scale, int accumulate,
                                                        float *__restrict__ part, float *__restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int cb = blockIdx.y * 4 * LPR * NCH;
  const int c = 4 * (lane % LPR), cols = d - cb;  // columns of this block, from cb
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const bool writer = lane < LPR;
  float acc[NCH][4];
  const T *base = drows + cb;
  if (wave < chunks) {
    const int p0 = static_cast<int>(wave) * ES_CHUNK, p1 = n - p0 < ES_CHUNK ? n : p0 + ES_CHUNK;
    const uint32_t k0 = keys[p0], k1 = keys[p1 - 1];
#pragma unroll 1
    for (int slot = 0; slot < 2; ++slot) {
      const uint32_t k = slot ? k1 : k0;
      if (k >= static_cast<uint32_t>(V) || (slot && k1 == k0)) continue;
      const Run run = runs[k];
      if (run.end - run.start <= ES_CHUNK) continue;
      const int a = run.start > p0 ? run.start : p0, b = run.end < p1 ? run.end : p1;
      sum_rows<T, LPR, NCH>(base, ld, rows, a, b, c, cols, acc);
      float *dst = part + (2 * wave + slot) * d + cb + c;
#pragma unroll
      for (int q = 0; q < NCH; ++q)
        if (writer) put4(dst + q * 4 * LPR, c + q * 4 * LPR, cols, acc[q], 1.f, false);
    }
    return;
  }
  const int64_t v = wave - chunks;
  if (v >= V) return;
  const Run run = runs[v];
  if (run.end - run.start > ES_CHUNK || (accumulate && run.end == run.start)) return;
  sum_rows<T, LPR, NCH>(base, ld, rows, run.start, run.end, c, cols, acc);
  float *dst = out + v * d + cb + c;
#pragma unroll
  for (int q = 0; q < NCH; ++q)
    if (writer) put4(dst + q * 4 * LPR, c + q * 4 * LPR, cols, acc[q], scale, accumulate != 0);
}

// Long runs: workgroup (chunk, column block of 64) owns the run that starts in its chunk and leaves it, if there is one
// (it holds the chunk's last position), and adds the run's partials in chunk order: 16 groups of 16 lanes take every
// 16th partial, then the groups are added in order.
__global__ __launch_bounds__(256) void embed_join_kernel(const uint32_t *__restrict__ keys, const Run *__restrict__ runs,
                                                         int32_t n, int32_t V, int d, const float *__restrict__ part,
                                                         float scale, int accumulate, float *__restrict__ out) {
  __shared__ float red[16][64];
  const int64_t p0 = static_cast<int64_t>(blockIdx.x) * ES_CHUNK;
  const int64_t p1 = p0 + ES_CHUNK < n ? p0 + ES_CHUNK : n;
  const uint32_t k = keys[p1 - 1];
  if (k >= static_cast<uint32_t>(V)) return;
  const Run run = runs[k];
  if (run.end - run.start <= ES_CHUNK || run.start < p0) return;
  const int64_t first = blockIdx.x, count = (run.end - 1) / ES_CHUNK - first + 1;
  const int64_t lead = 2 * first + (run.start == p0 ? 0 : 1);
  const int g = threadIdx.x >> 4, c = blockIdx.y * 64 + 4 * (threadIdx.x & 15);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t j = g; j < count; j += 16) {
    const float *src = part + (j == 0 ? lead : 2 * (first + j)) * d + c;
    if (c + 4 <= d) {
      float v[4];
      load_row<4>(src, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += v[e];
    } else {
      for (int e = 0; e < 4 && c + e < d; ++e) acc[e] += src[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) red[g][4 * (threadIdx.x & 15) + e] = acc[e];
  __syncthreads();
  if (threadIdx.x < 16) {
    float t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      t[e] = 0.f;
      for (int q = 0; q < 16; ++q) t[e] += red[q][4 * threadIdx.x + e];
    }
    if (c < d) put4(out + static_cast<int64_t>(k) * d + c, c, d, t, scale, accumulate != 0);
  }
}

struct SortPlan {
  int64_t keys[2], rows[2], runs, counts, totals, part, bytes;  // offsets in the workspace
  int passes, bits, tiles, chunks;
};

static SortPlan sort_plan(int64_t n, int32_t V, int32_t d) {
  SortPlan p = {};
  int64_t at = 0;
  auto take = [&](int64_t b) {
    const int64_t o = at;
    at += (b + 255) / 256 * 256;
    return o;
  };
  const bool rank = n <= ES_RANK_MAX;
  int need = 0;
  while ((static_cast<int64_t>(V) >> need) != 0) ++need;  // bits of the largest key, V
  p.passes = rank ? 0 : (need + ES_BITS - 1) / ES_BITS;
  p.bits = rank ? 0 : (need + p.passes - 1) / p.passes;
  p.tiles = static_cast<int>((n + ES_TILE - 1) / ES_TILE);
  p.chunks = n > ES_CHUNK ? static_cast<int>((n + ES_CHUNK - 1) / ES_CHUNK) : 0;  // no run of n <= 64 rows is long
  p.keys[0] = take(4 * n);
  p.rows[0] = take(4 * n);
  p.keys[1] = rank ? 0 : take(4 * n);
  p.rows[1] = rank ? 0 : take(4 * n);
  p.runs = take(static_cast<int64_t>(sizeof(Run)) * V);
  p.counts = rank ? 0 : take(static_cast<int64_t>(4) * p.tiles << p.bits);
  p.totals = rank ? 0 : take(int64_t(4) << p.bits);
  p.part = take(static_cast<int64_t>(8) * p.chunks * d);
  p.bytes = at;
  return p;
}

template <typename T>
static void launch_sum(const SortPlan &p, const T *drows, int64_t ld, int32_t n, int32_t V, int d, const uint32_t *keys,
                       const int32_t *rows, const Run *runs, float scale, int accumulate, float *part, float *out,
                       hipStream_t s) {
  const unsigned gx = static_cast<unsigned>((static_cast<int64_t>(p.chunks) + V + 3) / 4);
#define VK_EMBED_SUM(LPR, NCH)                                                                                          \
  embed_sum_kernel<T, LPR, NCH><<<dim3(gx, static_cast<unsigned>((d + 4 * LPR * NCH - 1) / (4 * LPR * NCH))), 256, 0, s>>>( \
      drows, ld, n, V, d, keys, rows, runs, p.chunks, scale, accumulate, part, out)
  if (d <= 64)
    VK_EMBED_SUM(16, 1);
  else if (d <= 128)
    VK_EMBED_SUM(32, 1);
  else if (d <= 256)
    VK_EMBED_SUM(64, 1);
  else if (d <= 512)
    VK_EMBED_SUM(64, 2);
  else if (d <= 768)
    VK_EMBED_SUM(64, 3);
  else
    VK_EMBED_SUM(64, 4);
#undef VK_EMBED_SUM
}

}  // namespace vk

using namespace vk;

extern "C" int vk_embed_lookup(const void *w, int32_t w_dtype, const int64_t *tokens, int64_t n, int64_t V, int32_t d,
                               float scale, void *out, int32_t out_dtype, void *stream) {
  VK_CHECK_ARG(n >= 0 && V > 0 && d > 0, "embed_lookup: bad sizes (V=%lld d=%d)", static_cast<long long>(V), d);
  VK_CHECK_ARG(n == 0 || (w && tokens && out), "embed_lookup: null pointer");
  VK_CHECK_ARG((w_dtype == VK_DTYPE_BF16 || w_dtype == VK_DTYPE_F32) && (out_dtype == VK_DTYPE_BF16 || out_dtype == VK_DTYPE_F32),
               "embed_lookup: bad dtype");
  if (n == 0) return VK_OK;
  const bool wf = w_dtype == VK_DTYPE_F32, of = out_dtype == VK_DTYPE_F32;
  const int per = !wf && !of ? 8 : 4;  // elements per lane
  const int lpr = d <= 16 * per ? 16 : (d <= 32 * per ? 32 : 64);
  const int64_t rows_per_block = 4 * EL_ROWS * (64 / lpr), blocks = (n + rows_per_block - 1) / rows_per_block;
  VK_CHECK_ARG(blocks < (int64_t(1) << 31), "embed_lookup: too many rows");
  hipStream_t s = VK_STREAM(stream);
#define VK_LOOKUP(WT, OT)                                                                                              \
  do {                                                                                                                 \
    auto k = lpr == 16 ? embed_lookup_kernel<WT, OT, 16> : (lpr == 32 ? embed_lookup_kernel<WT, OT, 32>                \
                                                                     : embed_lookup_kernel<WT, OT, 64>);               \
    k<<<static_cast<unsigned>(blocks), 256, 0, s>>>(static_cast<const WT *>(w), tokens, n, V, d, scale,                \
                                                    static_cast<OT *>(out));                                           \
  } while (0)
  if (wf && of)
    VK_LOOKUP(float, float);
  else if (wf)
    VK_LOOKUP(float, bf16_t);
  else if (of)
    VK_LOOKUP(bf16_t, float);
  else
    VK_LOOKUP(bf16_t, bf16_t);
#undef VK_LOOKUP
  return launch_status("embed_lookup");
}

extern "C" int vk_embed_grad_sorted_workspace(int64_t n, int32_t V, int32_t d, int64_t *bytes) {
  VK_CHECK_ARG(bytes && n >= 0 && V > 0 && d > 0, "embed_grad_sorted_workspace: bad arguments");
  VK_CHECK_ARG(n < (int64_t(1) << 31) - ES_TILE, "embed_grad_sorted: too many rows");
  *bytes = sort_plan(n, V, d).bytes;
  return VK_OK;
}

extern "C" int vk_embed_grad_sorted(const void *d_rows, int32_t d_dtype, int64_t ld, const int64_t *tokens, int64_t n,
                                    int32_t V, int32_t d, float scale, int64_t pad, float *out, int32_t accumulate,
                                    void *workspace, int64_t workspace_bytes, void *stream) {
  VK_CHECK_ARG(n >= 0 && V > 0 && d > 0 && ld >= d, "embed_grad_sorted: bad sizes (V=%d d=%d)", V, d);
  VK_CHECK_ARG(n < (int64_t(1) << 31) - ES_TILE, "embed_grad_sorted: too many rows");
  VK_CHECK_ARG(out && workspace && (n == 0 || (d_rows && tokens)), "embed_grad_sorted: null pointer");
  VK_CHECK_ARG(d_dtype == VK_DTYPE_BF16 || d_dtype == VK_DTYPE_F32, "embed_grad_sorted: bad row dtype");
  VK_CHECK_ARG(vk_aligned16(workspace), "embed_grad_sorted: workspace must be 16-byte aligned");
  const SortPlan p = sort_plan(n, V, d);
  VK_CHECK_ARG(workspace_bytes >= p.bytes, "embed_grad_sorted: workspace of %lld bytes needed",
               static_cast<long long>(p.bytes));
  hipStream_t s = VK_STREAM(stream);
  char *ws = static_cast<char *>(workspace);
  auto keys = [&](int i) { return reinterpret_cast<uint32_t *>(ws + p.keys[i]); };
  auto rows = [&](int i) { return reinterpret_cast<int32_t *>(ws + p.rows[i]); };
  Run *runs = reinterpret_cast<Run *>(ws + p.runs);
  int at = 0;  // which of the two key / row buffers holds the sorted ones
  if (p.passes == 0) {
    embed_runs_clear_kernel<<<static_cast<unsigned>((static_cast<int64_t>(V) + 255) / 256), 256, 0, s>>>(runs, V);
    if (n > 0)
      embed_rank_kernel<<<static_cast<unsigned>((n + ES_RANK_ROWS - 1) / ES_RANK_ROWS), 256, 0, s>>>(
          tokens, static_cast<int32_t>(n), V, pad, keys(0), rows(0), runs);
  } else {
    uint32_t *counts = reinterpret_cast<uint32_t *>(ws + p.counts), *totals = reinterpret_cast<uint32_t *>(ws + p.totals);
    const unsigned tiles = static_cast<unsigned>(p.tiles), bins = 1u << p.bits;
    for (int q = 0; q < p.passes; ++q) {
      const int shift = q * p.bits, to = q & 1;
      if (q == 0)
        embed_hist_kernel<true><<<tiles, 256, 0, s>>>(tokens, nullptr, n, V, pad, shift, bins, counts, runs);
      else
        embed_hist_kernel<false><<<tiles, 256, 0, s>>>(nullptr, keys(at), n, V, pad, shift, bins, counts, nullptr);
      embed_scan_kernel<<<bins, 64, 0, s>>>(counts, p.tiles, totals);
      if (q == 0)
        embed_scatter_kernel<true><<<tiles, 256, 0, s>>>(tokens, nullptr, nullptr, n, V, pad, shift, p.bits, counts,
                                                         totals, keys(to), rows(to));
      else
        embed_scatter_kernel<false><<<tiles, 256, 0, s>>>(nullptr, keys(at), rows(at), n, V, pad, shift, p.bits, counts,
                                                          totals, keys(to), rows(to));
      at = to;
    }
    embed_runs_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, s>>>(keys(at), n, V, runs);
  }
  int rc = launch_status("embed_grad_sorted sort");
  if (rc != VK_OK) return rc;
  float *part = reinterpret_cast<float *>(ws + p.part);
  if (d_dtype == VK_DTYPE_F32)
    launch_sum(p, static_cast<const float *>(d_rows), ld, static_cast<int32_t>(n), V, d, keys(at), rows(at), runs, scale,
               accumulate, part, out, s);
  else
    launch_sum(p, static_cast<const bf16_t *>(d_rows), ld, static_cast<int32_t>(n), V, d, keys(at), rows(at), runs, scale,
               accumulate, part, out, s);
  rc = launch_status("embed_grad_sorted sum");
  if (rc != VK_OK || p.chunks == 0) return rc;
  embed_join_kernel<<<dim3(static_cast<unsigned>(p.chunks), static_cast<unsigned>((d + 63) / 64)), 256, 0, s>>>(
      keys(at), runs, static_cast<int32_t>(n), V, d, part, scale, accumulate, out);
  return launch_status("embed_grad_sorted join");
}
