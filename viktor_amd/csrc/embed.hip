// The token embedding at vocabularies past the 4-mers': the lookup of scaled rows and the table's gradient.
//
// Lookup: out[r, :] = round(scale * W[t_r, :]), the product in fp32. Ids outside [0, V) give zero rows. Bound by the rows
// written (a frequent token's row is read from a cache: of 1074 MB gathered from an 11 MB table, 542 pass the L2s): 524288
// rows of 512 fp32 take 224 us (4.8 TB/s written), 40961 of 1000 bf16 24 us; with stores that go through the caches 244 and
// 31. The same 40961 from bf16 to fp32 44, fp32 to bf16 37, fp32 to fp32 47.5.
//
// Gradient: g[v, :] = scale * sum over t_r = v of dY[r, :], fp32, without atomics on floats. Rows are brought into token
// order first (a stable sort of the ids, row numbers as its payload), so that every vocabulary row is one run of
// consecutive sorted positions in ascending row order; the sum then reads each gradient row once, in an order that only
// n, V and the ids decide. Ids outside [0, V), and `pad`, get the key V: they sort behind every row and no sum reads
// them. The sort:
//   n <= ES_RANK_MAX: the position of a row is a count, pos = #{key_j < key_i} + #{j < i: key_j = key_i}, taken over all
//     n keys in LDS, in one launch;
//   larger n: radix passes over digits of at most 9 bits (2 for the vocabularies of k = 5 .. 8), each a histogram per tile
//     of 1024 or 2048 keys and a stable scatter.
// The sum goes by chunks of 16 to 64 sorted positions, one wavefront per 16 bytes x 64 columns of each, with the loads of 8
// gradient rows in flight whatever runs they belong to: it writes the runs that start in its chunk, up to a chunk past it.
// A longer run (padding, a homopolymer: tokens that a large part of the rows share) is cut at the chunks' borders, so that
// it spreads over the chip; the join adds its partial sums in chunk order. Rows without a run are zeroed by wavefronts of
// their own.
// What bounds it: few rows, the launches in series (1003 x 512 fp32: rank 4.4, sum 6.5, join 3.2 us); many, the sum's bytes
// (524288 x 512 fp32 into 87383 rows: 194 us for 1035 MB, 5.3 TB/s; the sort 36 us, the join 5.5). 98305 x 768 bf16 into
// 21847 rows: sort 22, sum 48 (218 MB), join 7.5.
#include "row_access.h"

namespace vk {

constexpr int EL_WIDTH_MAX = 1 << 20;                // elements of a row
constexpr int64_t EL_GRID_MAX = int64_t(1) << 24;  // workgroups of 256 threads: a launch has fewer than 2^32 threads

// LPR lanes share a row (64 / LPR rows per wavefront side by side), N elements each, as few as span the row (65536 bf16
// rows of 64, 128, 256: 4.5, 5.6, 9.1 us with 16, 16, 32 lanes, 10.8, 12.1, 12.7 with 64): 16-byte accesses of the narrower
// type where both are bf16, of the fp32 side otherwise. A group of columns that the row's end cuts is moved back to stay
// inside the row (columns that two lanes hold get the same value); rows narrower than a group go column by column. The
// rows written are not read again here: past the caches, which keep the table.
template <typename WT, typename OT, int LPR>
__global__ __launch_bounds__(256) void embed_lookup_kernel(const WT *__restrict__ w, const int64_t *__restrict__ tokens,
                                                           int64_t n, int64_t V, int d, float scale,
                                                           OT *__restrict__ out) {
  constexpr int N = sizeof(WT) + sizeof(OT) == 4 ? 8 : 4, SIDE = 64 / LPR;
  const int lane = threadIdx.x & 63, c0 = (lane % LPR) * N;
  const int64_t r = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * SIDE + lane / LPR;
  if (r >= n) return;
  const int64_t t = tokens[r];
  const bool in = t >= 0 && t < V;
  const WT *src = w + (in ? t : 0) * d;
  OT *dst = out + r * d;
  if (d < N) {
    for (int k = c0; k < d && k < c0 + N; ++k) store_one(dst + k, in ? load_one(src + k) * scale : 0.f);
    return;
  }
  for (int own = c0; own < d; own += LPR * N) {
    const int c = min(own, d - N);
    float v[N];
    load_row<N>(src + c, v);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = in ? v[k] * scale : 0.f;
    stream_out<N>(dst + c, v);
  }
}

// ---- the sort ----------------------------------------------------------------------------------------------------------

// The borders below, in rows, with the whole gradient's time on either side (us, rows of 512 fp32, 5463 ids).
// The counting sort up to here: its work grows with n^2. 2048 rows: 16.8, radix 23.4; 4096: 22.8, 24.6; 8192: 37.0, 27.1.
constexpr int ES_RANK_MAX = 4096;
constexpr int ES_RANK_ROWS = 16;  // rows per workgroup of it
// Tiles of 1024 keys up to here, which spread a pass over more CUs, then 2048, which make fewer tiles to sum. 32768 rows:
// 34.4, with 2048 36.8; 131072: 74.2, 74.6; 524288: 223 with 1024, 220.
constexpr int ES_SMALL = 131072;
constexpr int ES_BITS = 9;  // digit bits at most
// Tiles up to which a scatter sums the earlier tiles' counts itself, which spares a launch but reads all counts once per
// tile. 128 tiles (262144 rows of 64): 48.6, with a scan of its own 48.4; 256: 71.4, 68.8.
constexpr int ES_FUSED = 128;
// Chunks of 16 positions up to here: a wavefront's loads are serial, and few rows make few wavefronts. 1003 rows: 13.7, of
// 32 14.3, of 64 21.5; 16384: 29.0, 30.1, 35.3; 32768: 35.3, 34.2, 37.4.
constexpr int ES_SHORT = 16384;
// Chunks of 32 up to here, then 64: a chunk's border costs a long run a partial sum, written and read. 65536 rows: 52 with
// 16, 46.8 with 32, 48.3 with 64; 98304: 32 64.5, 64 64.1; 131072: 93, 74.5, 70.3; 262144: 190, 131, 117.
constexpr int ES_MEDIUM = 102400;

constexpr int64_t ES_ROWS_MAX = (int64_t(1) << 31) - 4096;  // (32-bit positions, a tile or chunk past the last included)
constexpr uint32_t ES_NONE = 0xffffffffu;  // a key that is none: ignored, or past the last

struct Pair {
  uint32_t key, row;
};

__device__ __forceinline__ uint32_t sort_key(int64_t t, int32_t V, int64_t pad) {
  return t >= 0 && t < V && t != pad ? static_cast<uint32_t>(t) : static_cast<uint32_t>(V);
}

// 16 rows per workgroup, 16 threads each over a sixteenth of the keys, four at a time. Bound by its n^2 / 4 LDS reads of 16
// bytes: 4.4 us at n = 1003.
__global__ __launch_bounds__(256) void embed_rank_kernel(const int64_t *__restrict__ tokens, int32_t n, int32_t V,
                                                         int64_t pad, Pair *__restrict__ sorted,
                                                         int32_t *__restrict__ owners) {
  __shared__ __attribute__((aligned(16))) uint32_t key[ES_RANK_MAX];
  if (blockIdx.x == 0 && threadIdx.x == 0) owners[0] = 0;
  const int up = (n + 3) & ~3;
  for (int j = threadIdx.x; j < up; j += 256) key[j] = j < n ? sort_key(tokens[j], V, pad) : ES_NONE;
  __syncthreads();
  const int part = threadIdx.x & 15;
  const int i = blockIdx.x * ES_RANK_ROWS + (threadIdx.x >> 4);
  const bool live = i < n;
  const uint32_t mine = key[live ? i : 0];
  int pos = 0;
#pragma unroll 4
  for (int j = 4 * part; j < up; j += 64) {
    const u32x4 k = *reinterpret_cast<const u32x4 *>(key + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) pos += k[e] < mine + (j + e < i ? 1u : 0u);  // smaller, or equal and earlier
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) pos += __shfl_xor(pos, o, 64);
  if (live && part == 0) sorted[pos] = Pair{mine, static_cast<uint32_t>(i)};
}

// counts [tiles, bins]: keys of each digit in each tile of KEYS x 1024 (4 to 5 us: a launch and one memory round trip).
// The first pass takes the ids themselves, and empties the list of long runs.
template <int KEYS, bool FIRST>
__global__ __launch_bounds__(1024) void embed_hist_kernel(const int64_t *__restrict__ tokens, const Pair *__restrict__ pairs,
                                                          int64_t n, int32_t V, int64_t pad, int shift, int bins,
                                                          uint32_t *__restrict__ counts, int32_t *__restrict__ owners) {
  if (FIRST && blockIdx.x == 0 && threadIdx.x == 0) owners[0] = 0;
  // four counters a digit, by lane: a digit that many keys share is not added to one place by a whole wavefront
  __shared__ u32x4 h[1 << ES_BITS];
  for (int b = threadIdx.x; b < bins; b += 1024) h[b] = u32x4{0u, 0u, 0u, 0u};
  const int64_t base = static_cast<int64_t>(blockIdx.x) * KEYS * 1024;
  uint32_t k[KEYS];
#pragma unroll
  for (int u = 0; u < KEYS; ++u) {
    const int64_t i = base + u * 1024 + threadIdx.x, at = i < n ? i : n - 1;
    k[u] = FIRST ? sort_key(tokens[at], V, pad) : pairs[at].key;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < KEYS; ++u)
    if (base + u * 1024 + threadIdx.x < n)
      atomicAdd(reinterpret_cast<uint32_t *>(h) + 4 * ((k[u] >> shift) & (bins - 1)) + (threadIdx.x & 3), 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += 1024)
    counts[static_cast<int64_t>(blockIdx.x) * bins + b] = (h[b][0] + h[b][1]) + (h[b][2] + h[b][3]);
}

__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t up = __shfl_up(v, o, 64);
    if (lane >= o) v += up;
  }
  return v;
}

// More than ES_FUSED tiles: one wavefront per digit; its column of counts becomes its exclusive prefix over the tiles,
// totals[digit] its sum.
__global__ __launch_bounds__(64) void embed_scan_kernel(uint32_t *__restrict__ counts, int64_t tiles, int bins,
                                                        uint32_t *__restrict__ totals) {
  uint32_t *col = counts + blockIdx.x;
  const int lane = threadIdx.x;
  uint32_t run = 0;
  for (int64_t t0 = 0; t0 < tiles; t0 += 64) {
    const uint32_t v = t0 + lane < tiles ? col[(t0 + lane) * bins] : 0;
    const uint32_t inc = wave_scan(v, lane);
    if (t0 + lane < tiles) col[(t0 + lane) * bins] = run + inc - v;
    run += __shfl(inc, 63, 64);
  }
  if (lane == 0) totals[blockIdx.x] = run;
}

// A stable scatter: wavefront w of a tile owns 64 KEYS keys side by side, in KEYS rounds of 64, so (w, round, lane) is
// the keys' order. In a round the lanes of one digit find each other by a ballot per digit bit; a key's rank is the
// digit's count in this wavefront's earlier rounds plus its lanes below. FUSED: the tile's offsets are summed here from
// the counts of all (at most ES_FUSED) tiles, two threads per digit. 7 us at 98305 rows, 8 at 524288: the chain of load,
// ranks, offsets and scattered stores.
template <int KEYS, bool FIRST, bool FUSED>
__global__ __launch_bounds__(1024) void embed_scatter_kernel(const int64_t *__restrict__ tokens,
                                                             const Pair *__restrict__ in, int64_t n, int32_t V, int64_t pad,
                                                             int shift, int bits, const uint32_t *__restrict__ counts,
                                                             const uint32_t *__restrict__ totals,
                                                             Pair *__restrict__ out) {
  constexpr int BINS = 1 << ES_BITS, WAVES = 16;
  __shared__ uint32_t wcount[WAVES][BINS];
  __shared__ uint32_t half[2][BINS], wsum[WAVES];
  const int bins = 1 << bits, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * KEYS * 1024 + wid * KEYS * 64;
  Pair x[KEYS];
#pragma unroll
  for (int r = 0; r < KEYS; ++r) {
    const int64_t i = base + r * 64 + lane, at = i < n ? i : n - 1;
    x[r] = FIRST ? Pair{sort_key(tokens[at], V, pad), static_cast<uint32_t>(i)} : in[at];
  }
  // this digit's keys in earlier tiles, and in all
  uint32_t before = 0, total = 0;
  const int bin = tid & (BINS - 1), side = tid / BINS;
  if (bin < bins) {
    if (FUSED) {
      const int tiles = static_cast<int>(gridDim.x), me = static_cast<int>(blockIdx.x);
      for (int t0 = side; t0 < tiles; t0 += 32) {
        uint32_t c[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) c[u] = counts[min(t0 + 2 * u, tiles - 1) * bins + bin];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          total += t0 + 2 * u < tiles ? c[u] : 0;
          before += t0 + 2 * u < me ? c[u] : 0;
        }
      }
    } else if (side == 0) {
      before = counts[static_cast<int64_t>(blockIdx.x) * bins + bin];
      total = totals[bin];
    }
  }
  for (int b = tid; b < WAVES * BINS; b += 1024) (&wcount[0][0])[b] = 0;
  if (side == 1) {
    half[0][bin] = before;
    half[1][bin] = total;
  }
  __syncthreads();
  if (FUSED && side == 0) {
    before += half[0][bin];
    total += half[1][bin];
  }
  int rank[KEYS];
  volatile uint32_t *mine = wcount[wid];
  const uint64_t below_mask = (uint64_t(1) << lane) - 1;
#pragma unroll
  for (int r = 0; r < KEYS; ++r) {
    const bool live = base + r * 64 + lane < n;
    const uint32_t dig = (x[r].key >> shift) & (bins - 1);
    uint64_t peers = __ballot(live);
#pragma unroll
    for (int b = 0; b < ES_BITS; ++b) {
      const bool bit = (dig >> b) & 1;
      const uint64_t m = __ballot(bit);
      if (b < bits) peers &= bit ? m : ~m;
    }
    const int below = __popcll(peers & below_mask);
    const uint32_t old = mine[dig];  // every lane reads before a digit's first lane writes (one wavefront, in order)
    rank[r] = static_cast<int>(old) + below;
    if (live && below == 0) mine[dig] = old + static_cast<uint32_t>(__popcll(peers));
  }
  // digits' first positions: a scan of the totals over threads 0 .. 511
  const uint32_t inc = wave_scan(side == 0 ? total : 0, lane);
  if (lane == 63) wsum[wid] = inc;
  __syncthreads();
  if (side == 0 && bin < bins) {
    uint32_t at = inc - total + before;
    for (int w = 0; w < wid; ++w) at += wsum[w];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const uint32_t c = wcount[w][bin];
      wcount[w][bin] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < KEYS; ++r)
    if (base + r * 64 + lane < n) out[wcount[wid][(x[r].key >> shift) & (bins - 1)] + rank[r]] = x[r];
}

// ---- the sums ----------------------------------------------------------------------------------------------------------

// The N columns of a lane in the sum. A group that the row's end cuts is moved back to stay inside the row, so that all
// accesses are 16 bytes wide (columns that two lanes hold get the same sum); `own` is where its own columns begin. PLAIN:
// sums are stored; else they may be added to what is there, and rows may be narrower than a group, column by column (the
// whole gradient, us, stored and added: 98305 x 768 bf16 into 21847 rows 78 and 134, fp32 105 and 134; 65536 x 512 fp32 into
// 5463 53 and 66; rows of 7 bf16 70 and 73, of 3 fp32 36.5 and 38).
template <typename T, bool PLAIN>
struct Cols {
  static constexpr int N = 16 / sizeof(T), SPAN = 64 * N, U = 8;
  int own, c, d;
  float v[N];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = 0.f;
  }
  __device__ __forceinline__ void init(int block, int lane, int d_) {
    d = d_;
    own = block * SPAN + N * lane;
    c = own + N <= d || (!PLAIN && d < N) ? own : d - N;
    zero();
  }
  __device__ __forceinline__ u32x4 load(const T *row) const {
    if (PLAIN || d >= N) return stream_16(row + c);
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if constexpr (sizeof(T) == 4)
        w[k] = __float_as_uint(own + k < d ? load_one(row + own + k) : 0.f);
      else
        w[k] = pack_bf(own + 2 * k < d ? load_one(row + own + 2 * k) : 0.f,
                       own + 2 * k + 1 < d ? load_one(row + own + 2 * k + 1) : 0.f);
    return w;
  }
  __device__ __forceinline__ void add(const u32x4 &w) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if constexpr (sizeof(T) == 4)
        v[k] += __uint_as_float(w[k]);
      else
        v[k] += (k & 1) ? hi_bf(w[k / 2]) : lo_bf(w[k / 2]);
  }
  // scale * the sums into a row (`onto`: added to it); the sums start over.
  __device__ __forceinline__ void put(float *row, float scale, bool onto) {
    if (own < d) {
      if (PLAIN || (!onto && d >= N)) {
        float o[N];
#pragma unroll
        for (int k = 0; k < N; ++k) o[k] = v[k] * scale;
        store_row<N>(row + c, o);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (c + k >= own && c + k < d) row[c + k] = onto ? row[c + k] + v[k] * scale : v[k] * scale;
      }
    }
    zero();
  }
  // Adds positions [a, b) of 64, whose gradient rows' numbers are in the lanes of `rows`: U rows' loads in flight. RUNS:
  // where `heads` has a bit, the run before that position ends; it goes to the row of `out` that its key names.
  template <bool RUNS>
  __device__ __forceinline__ void walk(const T *drows, int64_t ld, uint32_t rows, int a, int b, uint64_t heads,
                                       uint32_t keys, float *out, float scale, bool onto) {
    for (int p = a; p < b; p += U) {
      u32x4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = p + u < b ? p + u : b - 1;
        w[u] = load(drows + static_cast<int64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(rows, at))) * ld);
      }
      const uint32_t h = RUNS ? static_cast<uint32_t>(heads >> p) : 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p + u < b) {
          if (RUNS && ((h >> u) & 1))
            put(out + static_cast<int64_t>(__builtin_amdgcn_readlane(keys, p + u - 1)) * d, scale, onto);
          add(w[u]);
        }
      }
    }
  }
};

// Wavefronts 0 .. chunks - 1: the runs of a chunk of sorted positions, for the columns of block blockIdx.y. A run is long
// if it starts in a chunk and holds the last position of the next one: then its part in each chunk is a partial sum
// (slot 1: the one that starts there; slot 0: the one that comes in from the chunk before), and its first chunk goes on
// `owners`, in any order. The other wavefronts zero 64 vocabulary rows each, those without a run.
template <typename T, bool PLAIN, int CHUNK>
__global__ __launch_bounds__(256) void embed_sum_kernel(const T *__restrict__ drows, int64_t ld, int32_t n, int32_t V,
                                                        int d, const Pair *__restrict__ sorted, int32_t chunks, float scale,
                                                        int accumulate, float *__restrict__ part,
                                                        int32_t *__restrict__ owners, float *__restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t uV = static_cast<uint32_t>(V);
  Cols<T, PLAIN> x;
  x.init(blockIdx.y, lane, d);
  if (wave >= chunks) {
    const int64_t v0 = (wave - chunks) * 64, v = v0 + lane;
    if (v0 >= V || accumulate) return;
    int lo = 0, hi = n;  // first sorted position whose key is not below v
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (sorted[mid].key < static_cast<uint32_t>(v))
        lo = mid + 1;
      else
        hi = mid;
    }
    const bool absent = v < V && !(lo < n && sorted[lo].key == static_cast<uint32_t>(v));
    for (uint64_t left = __ballot(absent); left != 0; left &= left - 1)
      x.put(out + (v0 + __builtin_ctzll(left)) * d, 1.f, false);
    return;
  }
  const int p0 = static_cast<int>(wave) * CHUNK;
  auto at = [&](int p) {
    const Pair x = sorted[p < n ? p : n - 1];
    return Pair{p < n && x.key < uV ? x.key : ES_NONE, x.row};
  };
  constexpr uint64_t LANES = CHUNK == 64 ? ~uint64_t(0) : (uint64_t(1) << (CHUNK & 63)) - 1;
  const Pair lo = at(p0 + lane), hi = at(p0 + CHUNK + lane);
  const Pair before = at(p0 > 0 ? p0 - 1 : 0), before2 = at(p0 > CHUNK ? p0 - CHUNK - 1 : 0);
  const uint32_t prev = p0 > 0 ? before.key : ES_NONE, prev2 = p0 > CHUNK ? before2.key : ES_NONE;
  const int valid = __popcll(__ballot(lo.key != ES_NONE) & LANES);
  const uint32_t first = __builtin_amdgcn_readlane(lo.key, 0), last = __builtin_amdgcn_readlane(lo.key, CHUNK - 1);
  if (first == ES_NONE) return;
  uint32_t left_lo = __shfl_up(lo.key, 1, 64), left_hi = __shfl_up(hi.key, 1, 64);
  if (lane == 0) {
    left_lo = prev;
    left_hi = last;
  }
  const uint64_t heads = __ballot(lo.key != left_lo) & LANES, heads_hi = __ballot(hi.key != left_hi) & LANES;
  // [0, start): the run that comes in; [start, stop): this chunk's runs, of which the last goes on for `ahead` positions
  // of the next chunk; or [stop, CHUNK) is a long one
  const int start = heads != 0 ? __builtin_ctzll(heads) : CHUNK;
  const bool long_in = start > 0 && (prev2 == first || start == CHUNK);
  int ahead = last == ES_NONE || start == CHUNK ? 0 : (heads_hi != 0 ? __builtin_ctzll(heads_hi) : CHUNK);
  const bool long_out = ahead == CHUNK;
  const int stop = long_out ? 63 - __builtin_clzll(heads) : valid;
  const bool onto = accumulate != 0;
  if (long_in) {
    x.template walk<false>(drows, ld, lo.row, 0, start < valid ? start : valid, 0, 0, nullptr, 0.f, false);
    x.put(part + 2 * wave * d, 1.f, false);
  }
  if (start < stop) {
    x.template walk<true>(drows, ld, lo.row, start, stop, heads & ~(uint64_t(1) << start), lo.key, out, scale, onto);
    if (!long_out) x.template walk<false>(drows, ld, hi.row, 0, ahead, 0, 0, nullptr, 0.f, false);
    x.put(out + static_cast<int64_t>(__builtin_amdgcn_readlane(lo.key, stop - 1)) * d, scale, onto);
  }
  if (long_out) {
    x.template walk<false>(drows, ld, lo.row, stop, CHUNK, 0, 0, nullptr, 0.f, false);
    x.put(part + (2 * wave + 1) * d, 1.f, false);
    if (lane == 0 && blockIdx.y == 0) owners[1 + atomicAdd(owners, 1)] = static_cast<int32_t>(wave);
  }
}

constexpr int EJ_GROUPS = 32;

// Long runs: workgroups take (a run's first chunk, 64 columns) and add the run's partials in chunk order: 32 groups of 16
// lanes take every 32nd, then the groups are added in order. 3.2 us for a fifth of 1003 rows, 5.5 for one of 524288; a
// workgroup per chunk, most of which have nothing to add, took 115 us there.
__global__ __launch_bounds__(512) void embed_join_kernel(const Pair *__restrict__ sorted, int d, int chunk, int32_t chunks,
                                                         const float *__restrict__ part, const int32_t *__restrict__ owners,
                                                         float scale, int accumulate, float *__restrict__ out) {
  constexpr int U = 4;
  __shared__ float red[EJ_GROUPS][64];
  const int tid = threadIdx.x, g = tid >> 4, e0 = 4 * (tid & 15);
  const int blocks = (d + 63) / 64;
  const int64_t units = static_cast<int64_t>(owners[0]) * blocks;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int j = owners[1 + unit / blocks], c = static_cast<int>(unit % blocks) * 64 + e0;
    const uint32_t key = sorted[static_cast<int64_t>(j) * chunk + chunk - 1].key;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    bool more = true;
    for (int64_t i = j + g; more; i += U * EJ_GROUPS) {
      uint32_t k[U];
      float v[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t iu = i + u * EJ_GROUPS, in = iu < chunks ? iu : chunks - 1;
        k[u] = iu < chunks ? (iu == j ? key : sorted[in * chunk].key) : ES_NONE;
        const float *src = part + (2 * in + (iu == j ? 1 : 0)) * d;
        if (c + 4 <= d) {
          load_row<4>(src + c, v[u]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[u][e] = src[min(c + e, d - 1)];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        more = more && k[u] == key;  // (sorted: no later chunk begins with it then)
        if (more)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] += v[u][e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) red[g][e0 + e] = acc[e];
    __syncthreads();
    const int col = static_cast<int>(unit % blocks) * 64 + tid;
    if (tid < 64 && col < d) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < EJ_GROUPS; ++w) t += red[w][tid];
      float *dst = out + static_cast<int64_t>(key) * d + col;
      *dst = accumulate ? *dst + t * scale : t * scale;
    }
    __syncthreads();  // red has been read
  }
}

struct SortPlan {
  int64_t pairs[2], counts, totals, part, owners, bytes;  // offsets in the workspace
  int64_t tiles;
  int keys, passes, bits, chunk, chunks;
};

static SortPlan sort_plan(int64_t n, int32_t V, int32_t d) {
  SortPlan p = {};
  int64_t at = 0;
  auto take = [&](int64_t b) {
    const int64_t o = at;
    at += (b + 255) / 256 * 256;
    return o;
  };
  int need = 0;
  while ((static_cast<int64_t>(V) >> need) != 0) ++need;  // bits of the largest key, V
  p.passes = n <= ES_RANK_MAX ? 0 : (need + ES_BITS - 1) / ES_BITS;
  p.bits = p.passes == 0 ? 0 : (need + p.passes - 1) / p.passes;
  p.keys = n <= ES_SMALL ? 1 : 2;
  p.tiles = (n + p.keys * 1024 - 1) / (p.keys * 1024);
  p.chunk = n <= ES_SHORT ? 16 : (n <= ES_MEDIUM ? 32 : 64);
  p.chunks = static_cast<int>((n + p.chunk - 1) / p.chunk);
  p.pairs[0] = take(8 * n);
  p.pairs[1] = p.passes == 0 ? 0 : take(8 * n);
  p.counts = p.passes == 0 ? 0 : take((4 * p.tiles) << p.bits);
  p.totals = p.tiles <= ES_FUSED ? 0 : take(int64_t(4) << p.bits);
  p.part = n < 2 * p.chunk ? 0 : take(static_cast<int64_t>(8) * p.chunks * d);  // (no run is long in fewer)
  p.owners = take(4 * (p.chunks + 1));
  p.bytes = at < 16 ? 16 : at;
  return p;
}

template <int KEYS, bool FIRST>
static void launch_pass(const SortPlan &p, const int64_t *tokens, const Pair *in, Pair *out, int64_t n, int32_t V,
                        int64_t pad, int shift, uint32_t *counts, uint32_t *totals, int32_t *owners, hipStream_t s) {
  const unsigned tiles = static_cast<unsigned>(p.tiles), bins = 1u << p.bits;
  embed_hist_kernel<KEYS, FIRST><<<tiles, 1024, 0, s>>>(tokens, in, n, V, pad, shift, bins, counts, owners);
  if constexpr (KEYS == 2) {  // (1024 keys each: ES_SMALL rows are ES_FUSED tiles)
    if (p.tiles > ES_FUSED) {
      embed_scan_kernel<<<bins, 64, 0, s>>>(counts, p.tiles, bins, totals);
      embed_scatter_kernel<2, FIRST, false>
          <<<tiles, 1024, 0, s>>>(tokens, in, n, V, pad, shift, p.bits, counts, totals, out);
      return;
    }
  }
  static_assert(ES_SMALL <= 1024 * ES_FUSED, "tiles of 1024 keys have no scan of their own");
  embed_scatter_kernel<KEYS, FIRST, true><<<tiles, 1024, 0, s>>>(tokens, in, n, V, pad, shift, p.bits, counts, nullptr, out);
}

}  // namespace vk

using namespace vk;

extern "C" int vk_embed_lookup(const void *w, int32_t w_dtype, const int64_t *tokens, int64_t n, int64_t V, int32_t d,
                               float scale, void *out, int32_t out_dtype, void *stream) {
  VK_CHECK_ARG(n >= 0 && V > 0 && d > 0 && d <= EL_WIDTH_MAX, "embed_lookup: bad sizes (V=%lld d=%d)",
               static_cast<long long>(V), d);
  VK_CHECK_ARG(n == 0 || (w && tokens && out), "embed_lookup: null pointer");
  VK_CHECK_ARG((w_dtype == VK_DTYPE_BF16 || w_dtype == VK_DTYPE_F32) &&
                   (out_dtype == VK_DTYPE_BF16 || out_dtype == VK_DTYPE_F32),
               "embed_lookup: bad dtype");
  if (n == 0) return VK_OK;
  const bool wf = w_dtype == VK_DTYPE_F32, of = out_dtype == VK_DTYPE_F32;
  const int per = !wf && !of ? 8 : 4;  // elements per lane
  const int lpr = d <= 16 * per ? 16 : (d <= 32 * per ? 32 : 64);
  const int64_t rows_per_block = 4 * (64 / lpr), most = rows_per_block * (EL_GRID_MAX - 1);  // rows of a launch
  hipStream_t s = VK_STREAM(stream);
#define VK_LOOKUP(WT, OT)                                                                                              \
  do {                                                                                                                 \
    auto k = lpr == 16 ? embed_lookup_kernel<WT, OT, 16> : (lpr == 32 ? embed_lookup_kernel<WT, OT, 32>                \
                                                                     : embed_lookup_kernel<WT, OT, 64>);               \
    for (int64_t r = 0; r < n; r += most) {                                                                            \
      const int64_t rows = n - r < most ? n - r : most;                                                                \
      k<<<static_cast<unsigned>((rows + rows_per_block - 1) / rows_per_block), 256, 0, s>>>(                           \
          static_cast<const WT *>(w), tokens + r, rows, V, d, scale, static_cast<OT *>(out) + r * d);                  \
    }                                                                                                                  \
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
  VK_CHECK_ARG(bytes && n >= 0 && V > 0 && d > 0 && d <= EL_WIDTH_MAX, "embed_grad_sorted_workspace: bad arguments");
  VK_CHECK_ARG(n < ES_ROWS_MAX, "embed_grad_sorted: too many rows");
  *bytes = sort_plan(n, V, d).bytes;
  return VK_OK;
}

extern "C" int vk_embed_grad_sorted(const void *d_rows, int32_t d_dtype, int64_t ld, const int64_t *tokens, int64_t n,
                                    int32_t V, int32_t d, float scale, int64_t pad, float *out, int32_t accumulate,
                                    void *workspace, int64_t workspace_bytes, void *stream) {
  VK_CHECK_ARG(n >= 0 && V > 0 && d > 0 && d <= EL_WIDTH_MAX && ld >= d, "embed_grad_sorted: bad sizes (V=%d d=%d)", V, d);
  VK_CHECK_ARG(n < ES_ROWS_MAX, "embed_grad_sorted: too many rows");
  VK_CHECK_ARG(out && workspace && (n == 0 || (d_rows && tokens)), "embed_grad_sorted: null pointer");
  VK_CHECK_ARG(d_dtype == VK_DTYPE_BF16 || d_dtype == VK_DTYPE_F32, "embed_grad_sorted: bad row dtype");
  VK_CHECK_ARG(vk_aligned16(workspace), "embed_grad_sorted: workspace must be 16-byte aligned");
  const SortPlan p = sort_plan(n, V, d);
  VK_CHECK_ARG(workspace_bytes >= p.bytes, "embed_grad_sorted: workspace of %lld bytes needed",
               static_cast<long long>(p.bytes));
  const int64_t waves = p.chunks + (accumulate ? 0 : (static_cast<int64_t>(V) + 63) / 64);
  hipStream_t s = VK_STREAM(stream);
  char *ws = static_cast<char *>(workspace);
  auto pairs = [&](int i) { return reinterpret_cast<Pair *>(ws + p.pairs[i]); };
  int32_t *owners = reinterpret_cast<int32_t *>(ws + p.owners);
  int at = 0;  // which of the two buffers holds the sorted pairs
  if (n > 0 && p.passes == 0) {
    embed_rank_kernel<<<static_cast<unsigned>((n + ES_RANK_ROWS - 1) / ES_RANK_ROWS), 256, 0, s>>>(
        tokens, static_cast<int32_t>(n), V, pad, pairs(0), owners);
  } else if (n > 0) {
    uint32_t *counts = reinterpret_cast<uint32_t *>(ws + p.counts), *totals = reinterpret_cast<uint32_t *>(ws + p.totals);
    auto pass = p.keys == 1 ? launch_pass<1, true> : launch_pass<2, true>;
    pass(p, tokens, nullptr, pairs(0), n, V, pad, 0, counts, totals, owners, s);
    pass = p.keys == 1 ? launch_pass<1, false> : launch_pass<2, false>;
    for (int q = 1; q < p.passes; ++q) {
      pass(p, nullptr, pairs(at), pairs(1 - at), n, V, pad, q * p.bits, counts, totals, owners, s);
      at = 1 - at;
    }
  }
  int rc = launch_status("embed_grad_sorted sort");
  if (rc != VK_OK) return rc;
  float *part = reinterpret_cast<float *>(ws + p.part);
  if (waves == 0) return VK_OK;
  const unsigned gx = static_cast<unsigned>((waves + 3) / 4);  // (below EL_GRID_MAX by the limits of n and V)
#define VK_EMBED_SUM(T, PLAIN)                                                                                         \
  do {                                                                                                                 \
    auto k = p.chunk == 16 ? embed_sum_kernel<T, PLAIN, 16>                                                            \
                           : (p.chunk == 32 ? embed_sum_kernel<T, PLAIN, 32> : embed_sum_kernel<T, PLAIN, 64>);        \
    constexpr int span = Cols<T, PLAIN>::SPAN;                                                                         \
    k<<<dim3(gx, static_cast<unsigned>((d + span - 1) / span)), 256, 0, s>>>(                                          \
        static_cast<const T *>(d_rows), ld, static_cast<int32_t>(n), V, d, pairs(at), p.chunks, scale, accumulate, part, \
        owners, out);                                                                                                  \
  } while (0)
  const bool plain = !accumulate && d >= 8;
  if (d_dtype == VK_DTYPE_BF16 && plain)
    VK_EMBED_SUM(bf16_t, true);
  else if (d_dtype == VK_DTYPE_BF16)
    VK_EMBED_SUM(bf16_t, false);
  else if (plain)
    VK_EMBED_SUM(float, true);
  else
    VK_EMBED_SUM(float, false);
#undef VK_EMBED_SUM
  rc = launch_status("embed_grad_sorted sum");
  if (rc != VK_OK || n < 2 * p.chunk) return rc;
  const int64_t most = (n / (p.chunk + 1) + 1) * ((d + 63) / 64);  // (a long run: chunk + 1 rows)
  const int64_t cap = 4 * device_cus_cached();
  embed_join_kernel<<<static_cast<unsigned>(most < cap ? most : cap), 512, 0, s>>>(
      pairs(at), d, p.chunk, p.chunks, part, owners, scale, accumulate, out);
  return launch_status("embed_grad_sorted join");
}
