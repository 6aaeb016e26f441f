// Rows of a table by ids, scaled (f2c_embedding), and the table's gradient (f2c_embedding_backward).
//
// The lookup is bound by reading and writing the rows (121,000 x 128 float32 of 2.4 M rows: 18 us, 6.8 TB/s).  The gradient of row r is the sum of dy over
// the places i with ids[i] = r, in their order: the places are sorted by id (stable), every warp adds up a stretch of them, and a segment that lies in
// several stretches is put together by a last launch.  No atomics on values: the same bits every time.  Sums are single precision, rounded once.
//
// Up to 1024 places it is one launch (few_kernel): every CTA sorts all of them, in registers and shared memory, and adds up its share of the segments; what
// was not looked up is set to zero on the way.  (1024 places of 172 rows, 128 columns: 8.3 us in a graph, 7 in a row of calls; with
// the launches below 8.3 and 12.4 (rows alone), and 19 in a row of calls, whose launches the host makes.)
//
// More places of few rows (labels): a CTA sorts 400 places at most while their rows of dy come to its shared memory, and leaves a sum for every row of the table
// that it met; a second launch adds those up in the CTAs' order.  59,000 x 128 of 172 rows: 13.4 us (rows alone 19.5); all places sorted, from
// 59,201 of them on, 18.2 (26.7).
//
// Sorting.  Up to 4096 places each place counts the ones in front of it, in one launch: the keys are few enough that all pairs cost
// less than further launches.  Beyond, digits of up to 11 bits from the lowest on: counts of every tile of 1024 places, their sums over tiles, and the
// placing, in which a warp ranks 32 places at a time by their equals in it and counts the next digit where the places go.  As many digits as the table
// has rows need.  All of it is latency, 3 to 6 us a launch: the first one also clears what the others add to, and a whole table's gradient, on CTAs of its
// own.  (With tiles of 4096 places that add up the other tiles' counts themselves, two launches less, 121,000 places took 62 us instead of 51: the work
// was on too few SMs.)  121,000 places of 2.4 M rows, 128 columns, the rows alone: 51 us in eight launches (57 beside a lookup), 32 of
// them the sorting; the whole table in seven 256 us, of which clearing it is 168.
#include <algorithm>

#include "checkpoint.cuh"

namespace f2c {
namespace emb {

using ckpt::both;
using ckpt::f32x2;
using ckpt::Four;
using ckpt::kGroup;
using ckpt::mul2;
using ckpt::pair_of;
using ckpt::plus2;

constexpr int kThreads = 256, kWarps = kThreads / 32, kAhead = 4;
constexpr int64_t kMaxRows = (1ll << 31) - 2, kMaxPlaces = 1ll << 30, kMaxColumns = 1 << 20;

// ---------------------------------------------------------------- lookup
// A thread has kAhead vectors of ACCESS bytes of the result, all loads before the first use.
template <typename T, typename I, int ACCESS>
__global__ void __launch_bounds__(kThreads) lookup_kernel(const T* __restrict__ table, int64_t ld, int64_t rows, int vectors, const I* __restrict__ ids, int64_t m, float scale,
                                                          T* __restrict__ out) {
  constexpr int V = ACCESS / (int)sizeof(T);
  struct alignas(ACCESS) Vec { T v[V]; };
  dependency_wait();
  release_dependents();
  const int64_t first = (int64_t)blockIdx.x * (kThreads * kAhead), row0 = first / vectors;
  const uint32_t rest = (uint32_t)(first - row0 * vectors) + threadIdx.x;
  Vec v[kAhead];
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    const uint32_t at = rest + a * kThreads;
    const int64_t row = row0 + at / (uint32_t)vectors;
    const int64_t id = row < m ? (int64_t)__ldg(ids + row) : -1;
#pragma unroll
    for (int e = 0; e < V; ++e) v[a].v[e] = from_float<T>(0.0f);
    if ((uint64_t)id < (uint64_t)rows) v[a] = *(reinterpret_cast<const Vec*>(table + id * ld) + at % (uint32_t)vectors);
  }
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    const int64_t row = row0 + (rest + a * kThreads) / (uint32_t)vectors;
    if (row >= m) return;
#pragma unroll
    for (int e = 0; e < V; ++e) v[a].v[e] = from_float<T>(to_float(v[a].v[e]) * scale);
    *(reinterpret_cast<Vec*>(out) + first + threadIdx.x + a * kThreads) = v[a];
  }
}

// ---------------------------------------------------------------- sorting
constexpr int kItems = 4, kTile = kThreads * kItems, kMaxBits = 11, kFew = 4096;

// A row's number, or the number of rows where the id is outside the table.
template <typename I>
__device__ __forceinline__ uint32_t key_of(const I* ids, int64_t i, uint32_t rows) {
  const int64_t id = (int64_t)__ldg(ids + i);
  return (uint64_t)id < (uint64_t)rows ? (uint32_t)id : rows;
}

struct Pairs { uint32_t *key, *place; };

// Memory that the first launch sets to zero on its CTAs behind the others, 16 bytes at a time: `whole` of them from a 16-byte boundary on, and single
// bytes in front of and behind them.
struct Clear {
  uint8_t* at;
  int64_t front, whole, behind;
};
struct Clears { Clear of[2]; };
constexpr int kClearEach = 16;  // 16-byte words a thread
__device__ __forceinline__ void clear(const Clears& c, int64_t cta, int64_t ctas) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const Clear& m = c.of[q];
    uint4* const from = reinterpret_cast<uint4*>(m.at + m.front);
    for (int64_t i = cta * kThreads + threadIdx.x; i < m.whole; i += ctas * kThreads) from[i] = make_uint4(0u, 0u, 0u, 0u);
    if (cta == 0 && threadIdx.x < m.front) m.at[threadIdx.x] = 0;
    if (cta == 0 && threadIdx.x < m.behind) m.at[m.front + 16 * m.whole + threadIdx.x] = 0;
  }
}

// Few places: a warp finds the ranks of four at a time.
template <typename I>
__global__ void __launch_bounds__(kThreads) rank_kernel(const I* __restrict__ ids, int m, uint32_t rows, Pairs out, int ctas, const __grid_constant__ Clears zero) {
  __shared__ uint32_t keys[kFew];
  dependency_wait();
  release_dependents();
  if ((int)blockIdx.x >= ctas) return clear(zero, blockIdx.x - ctas, gridDim.x - ctas);
  for (int i = threadIdx.x; i < m; i += kThreads) keys[i] = key_of(ids, i, rows);
  __syncthreads();
  const int lane = threadIdx.x & 31, first = (blockIdx.x * kWarps + (threadIdx.x >> 5)) * 4;
  uint32_t mine[4];
  int before[4] = {};
#pragma unroll
  for (int q = 0; q < 4; ++q) mine[q] = keys[min(first + q, m - 1)];
  for (int j = lane; j < m; j += 32) {
    const uint32_t k = keys[j];
#pragma unroll
    for (int q = 0; q < 4; ++q) before[q] += k < mine[q] || (k == mine[q] && j < first + q);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int rank = __reduce_add_sync(0xffffffffu, before[q]);
    if (lane == 0 && first + q < m) {
      out.key[rank] = mine[q];
      out.place[rank] = (uint32_t)(first + q);
    }
  }
}

struct Digit { int shift, bits; };
__device__ __forceinline__ uint32_t digit_of(uint32_t key, Digit d) { return (key >> d.shift) & ((1u << d.bits) - 1u); }

// counts [tile][digit] of the first digit
template <typename I>
__global__ void __launch_bounds__(kThreads) count_kernel(const I* __restrict__ ids, int64_t m, uint32_t rows, Digit d, uint32_t* __restrict__ counts, int tiles,
                                                         const __grid_constant__ Clears zero) {
  __shared__ uint32_t here[1 << kMaxBits];
  dependency_wait();
  release_dependents();
  if ((int)blockIdx.x >= tiles) return clear(zero, blockIdx.x - tiles, gridDim.x - tiles);
  uint32_t key[kItems];
  const int64_t first = (int64_t)blockIdx.x * kTile + threadIdx.x;
#pragma unroll
  for (int q = 0; q < kItems; ++q) key[q] = first + q * kThreads < m ? key_of(ids, first + q * kThreads, rows) : 0u;
  for (int b = threadIdx.x; b < 1 << d.bits; b += kThreads) here[b] = 0u;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kItems; ++q)
    if (first + q * kThreads < m) atomicAdd(here + digit_of(key[q], d), 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < 1 << d.bits; b += kThreads) counts[((int64_t)blockIdx.x << d.bits) + b] = here[b];
}

// A digit to a lane: its counts become those of the tiles in front, and their sum goes to `totals`.  Each of the CTA's warps has a stretch of the tiles.
constexpr int kScanWarps = 32;
__global__ void __launch_bounds__(32 * kScanWarps) tiles_kernel(uint32_t* __restrict__ counts, uint32_t* __restrict__ totals, int tiles, int bins) {
  __shared__ uint32_t sums[kScanWarps][32];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bin = blockIdx.x * 32 + lane, each = (tiles + kScanWarps - 1) / kScanWarps;
  const int from = min(tiles, warp * each), to = min(tiles, from + each);
  uint32_t own = 0u;
  if (bin < bins) {
#pragma unroll 4
    for (int t = from; t < to; ++t) own += counts[(int64_t)t * bins + bin];
  }
  sums[warp][lane] = own;
  __syncthreads();
  uint32_t before = 0u, all = 0u;
#pragma unroll
  for (int w = 0; w < kScanWarps; ++w) {
    const uint32_t v = sums[w][lane];
    if (w < warp) before += v;
    all += v;
  }
  if (bin >= bins) return;
#pragma unroll 4
  for (int t = from; t < to; ++t) {
    uint32_t* const at = counts + (int64_t)t * bins + bin;
    const uint32_t v = *at;
    *at = before;
    before += v;
  }
  if (warp == 0) totals[bin] = all;
}

// `mine` of every thread becomes the sum of those of the threads in front.
__device__ __forceinline__ uint32_t block_before(uint32_t mine, uint32_t* of_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) of_warp[warp] = sum;
  __syncthreads();
  uint32_t before = sum - mine;
#pragma unroll
  for (int w = 0; w < kWarps; ++w)
    if (w < warp) before += of_warp[w];
  return before;
}

// Puts a tile's places where the digit wants them; counts_next (null: none): counts of the next digit, of the tiles in which they end up.
template <typename I, bool FIRST>
__global__ void __launch_bounds__(kThreads) place_kernel(const I* __restrict__ ids, Pairs in, int64_t m, uint32_t rows, Digit d, const uint32_t* __restrict__ counts,
                                                         const uint32_t* __restrict__ totals, Pairs out, Digit next, uint32_t* __restrict__ counts_next) {
  constexpr int kBins = 1 << kMaxBits, kEach = kBins / kThreads;
  __shared__ __align__(16) uint16_t of_warp[kWarps][kBins];  // a tile has 1024 places
  __shared__ __align__(16) uint32_t base[kBins];
  __shared__ uint32_t sums[kWarps];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = 1 << d.bits;
  uint32_t key[kItems], place[kItems], rank[kItems];
  const int64_t first = (int64_t)blockIdx.x * kTile + warp * (32 * kItems) + lane;
#pragma unroll
  for (int q = 0; q < kItems; ++q) {
    const int64_t i = first + 32 * q;
    key[q] = i < m ? (FIRST ? key_of(ids, i, rows) : in.key[i]) : 0u;
    place[q] = i < m ? (FIRST ? (uint32_t)i : in.place[i]) : 0u;
  }
  // where each digit's places of this tile start: eight digits (or as many as there are for everyone) a thread
  const int each = bins >= kBins ? kEach : (bins + kThreads - 1) / kThreads;
  uint32_t all[kEach], here[kEach], sum = 0u;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int b = threadIdx.x * each + e;
    const bool mine = e < each && b < bins;
    all[e] = mine ? __ldg(totals + b) : 0u;
    here[e] = mine ? __ldg(counts + ((int64_t)blockIdx.x << d.bits) + b) : 0u;
    sum += all[e];
  }
  for (int b = lane; b < bins / 2; b += 32) reinterpret_cast<uint32_t*>(of_warp[warp])[b] = 0u;  // (two digits at least)
  uint32_t before = block_before(sum, sums);
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const int b = threadIdx.x * each + e;
    if (e < each && b < bins) base[b] = before + here[e];
    before += all[e];
  }
#pragma unroll
  for (int q = 0; q < kItems; ++q) {
    const bool there = first + 32 * q < m;
    const uint32_t digit = digit_of(key[q], d), those = __ballot_sync(0xffffffffu, there);
    // the lanes with the same digit, bit by bit
    uint32_t equal = those;
#pragma unroll
    for (int b = 0; b < kMaxBits; ++b) {
      const bool one = (digit >> b) & 1u;
      const uint32_t ones = __ballot_sync(0xffffffffu, one);
      equal &= one ? ones : ~ones;
    }
    const uint32_t so_far = there ? of_warp[warp][digit] : 0u;
    __syncwarp();
    if (there && (equal & ((1u << lane) - 1u)) == 0u) of_warp[warp][digit] = (uint16_t)(so_far + __popc(equal));
    __syncwarp();
    rank[q] = so_far + __popc(equal & ((1u << lane) - 1u));
  }
  __syncthreads();
  for (int b = threadIdx.x; b < bins / 2; b += kThreads) {  // two digits at once: their sums over the tile's warps stay below 2^16
    uint32_t so_far = 0u;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      uint32_t* const at = reinterpret_cast<uint32_t*>(of_warp[w]) + b;
      const uint32_t own = *at;
      *at = so_far;
      so_far += own;
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kItems; ++q)
    if (first + 32 * q < m) {
      const uint32_t digit = digit_of(key[q], d), to = base[digit] + of_warp[warp][digit] + rank[q];
      out.key[to] = key[q];
      out.place[to] = place[q];
      if (counts_next != nullptr) atomicAdd(counts_next + ((int64_t)(to / kTile) << next.bits) + digit_of(key[q], next), 1u);
    }
}

// ---------------------------------------------------------------- sums over segments
// Stretches of up to 32 sorted places, a warp's each.
struct Segments {
  const uint32_t *key, *place;  // sorted
  int64_t m;
  uint32_t rows;                // keys of places without a row
  int stretch;                  // 8 to 32
  int64_t stretches;
  // only the rows that were looked up: numbers of segments in front of a stretch in its tile, and of those that begin in each tile, or (summed) in the tiles in front of each
  // and, last, in all of them
  const uint32_t *in_tile, *of_tile;
  int tiles;
  bool summed;
  int64_t* looked_up;           // null: the whole table
  int64_t* count;
};

// Whether a segment begins at sorted place i.
__device__ __forceinline__ bool begins(const uint32_t* key, int64_t i, int64_t m, uint32_t rows) {
  return i < m && key[i] < rows && (i == 0 || key[i - 1] != key[i]);
}

// Numbers the segments: a CTA to a tile of 1024 places.
__global__ void __launch_bounds__(kThreads) number_kernel(const uint32_t* __restrict__ key, int64_t m, uint32_t rows, int stretch, uint32_t* __restrict__ in_tile,
                                                          uint32_t* __restrict__ of_tile, int64_t* __restrict__ looked_up) {
  __shared__ uint32_t sums[kWarps];
  dependency_wait();
  release_dependents();
  const int64_t first = (int64_t)blockIdx.x * kTile + threadIdx.x * kItems;
  uint32_t own = 0u;
#pragma unroll
  for (int q = 0; q < kItems; ++q) {
    own += begins(key, first + q, m, rows);
    if (first + q < m) looked_up[first + q] = -1;  // (those that there are are written by the next launch)
  }
  const uint32_t before = block_before(own, sums);
  // a thread's four places are a part of one stretch
  if (first < m && first % stretch == 0) in_tile[first / stretch] = before;
  if (threadIdx.x == kThreads - 1) of_tile[blockIdx.x] = before + own;
}

// Beyond kTilesEach tiles their numbers are summed once, by a CTA; up to there every warp does so for itself, which saves a launch.  (Always so it was quadratic in the places:
// 2^24 of them, 8 columns, took 7.1 ms and 2.7 this way; 2^20 176 us and 164; 2^19 98 and 96, and 128 columns 148 and 149.)
constexpr int kTilesEach = 256, kSumThreads = 1024;
__global__ void __launch_bounds__(kSumThreads) sum_kernel(uint32_t* __restrict__ of_tile, int tiles) {
  __shared__ uint32_t of_warp[kSumThreads / 32];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, each = (tiles + kSumThreads - 1) / kSumThreads, from = min(tiles, (int)threadIdx.x * each), to = min(tiles, from + each);
  uint32_t own = 0u;
  for (int t = from; t < to; ++t) own += of_tile[t];
  uint32_t before = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) of_warp[warp] = before;
  __syncthreads();
  before = before - own + __reduce_add_sync(0xffffffffu, lane < warp ? of_warp[lane] : 0u);
  for (int t = from; t < to; ++t) {
    const uint32_t v = of_tile[t];
    of_tile[t] = before;
    before += v;
  }
  if (threadIdx.x == kSumThreads - 1) of_tile[tiles] = before;
}

constexpr int kRowsAhead = 8;

// What a stretch leaves: sums of the segment that it only continues (head) and of the one that goes on behind it (tail), and the tail's row (-1: none).
struct Open {
  float *head, *tail;  // [stretches][width]
  int64_t* row;        // [stretches]
  int64_t width;
};

template <typename T, int ACCESS>
__global__ void __launch_bounds__(kThreads) segment_kernel(const T* __restrict__ dy, int64_t ld, int d, float scale, const __grid_constant__ Segments s, const __grid_constant__ Open open,
                                                           T* __restrict__ out) {
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t c = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (c >= s.stretches) return;
  const int64_t start = c * s.stretch;
  const int n = (int)min((int64_t)s.stretch, s.m - start), col = blockIdx.y * kGroup + 4 * lane, left = d - col;
  const uint32_t key = lane < n ? s.key[start + lane] : s.rows, place = lane < n ? s.place[start + lane] : 0u;
  const uint32_t above = __shfl_up_sync(0xffffffffu, key, 1);
  const uint32_t before = lane == 0 && start > 0 ? s.key[start - 1] : s.rows;
  const uint32_t behind = start + n < s.m ? s.key[start + n] : s.rows;
  const uint32_t first = __ballot_sync(0xffffffffu, lane < n && (lane == 0 ? start == 0 || before != key : above != key));
  const int kept = __popc(__ballot_sync(0xffffffffu, key < s.rows));  // the places of no row are behind all others
  uint32_t row = key;  // of the result, for this lane's place (not where its segment begins in another stretch)
  if (s.looked_up != nullptr) {
    uint32_t tiles_before = 0u, all = 0u;
    const int tile = (int)(start / kTile);
    if (s.summed) {
      tiles_before = s.of_tile[tile];
      all = s.of_tile[s.tiles];
    } else {
      for (int t = lane; t < s.tiles; t += 32) {
        const uint32_t v = s.of_tile[t];
        all += v;
        if (t < tile) tiles_before += v;
      }
      all = __reduce_add_sync(0xffffffffu, all);
      tiles_before = __reduce_add_sync(0xffffffffu, tiles_before);
    }
    row = tiles_before + s.in_tile[c] + __popc(first & (0xffffffffu >> (31 - lane))) - 1u;
    if (blockIdx.y == 0) {
      if (c == 0 && lane == 0) *s.count = all;
      if (key < s.rows && ((first >> lane) & 1u)) s.looked_up[row] = (int64_t)key;
    }
    // rows behind the last segment's are zero
    for (int64_t r = max(start, (int64_t)all); r < start + n; ++r) {
      Four<T, ACCESS> zero;
      const f32x2 none[2] = {};
      zero.set(none);
      zero.store(out + r * d + col, left);
    }
  }
  f32x2 acc[2] = {};
  bool head = (first & 1u) == 0u;
  const auto write = [&](int last) {  // the segment whose last place here is `last`, and which ends there
    if (head) {
      *reinterpret_cast<ulonglong2*>(open.head + c * open.width + blockIdx.y * kGroup + 4 * lane) = make_ulonglong2(acc[0], acc[1]);
    } else {
      acc[0] = mul2(acc[0], both(scale));
      acc[1] = mul2(acc[1], both(scale));
      Four<T, ACCESS> v;
      v.set(acc);
      v.store(out + (int64_t)__shfl_sync(0xffffffffu, row, last) * d + col, left);
    }
    head = false;
    acc[0] = acc[1] = 0ull;
  };
  for (int t0 = 0; t0 < kept; t0 += kRowsAhead) {
    Four<T, ACCESS> v[kRowsAhead];
#pragma unroll
    for (int q = 0; q < kRowsAhead; ++q) {
      const int64_t at = __shfl_sync(0xffffffffu, place, (t0 + q) & 31);
      v[q].load(dy + at * ld + col, t0 + q < kept ? left : 0);
    }
#pragma unroll
    for (int q = 0; q < kRowsAhead; ++q) {
      const int t = t0 + q;
      if (t >= kept) break;
      if (t > 0 && ((first >> t) & 1u)) write(t - 1);
      f32x2 f[2];
      v[q].get(f);
      acc[0] = plus2(acc[0], f[0]);
      acc[1] = plus2(acc[1], f[1]);
    }
  }
  // the last segment may go on in the next stretch
  const bool opened = kept == n && !head && behind == __shfl_sync(0xffffffffu, key, n - 1);
  const int64_t opened_row = opened ? (int64_t)__shfl_sync(0xffffffffu, row, n - 1) : -1;
  if (opened) *reinterpret_cast<ulonglong2*>(open.tail + c * open.width + blockIdx.y * kGroup + 4 * lane) = make_ulonglong2(acc[0], acc[1]);
  else if (kept > 0) write(kept - 1);
  if (lane == 0 && blockIdx.y == 0) open.row[c] = opened_row;
}

// Puts the segments together that lie in several stretches: the tail of the one in which they begin, then heads.  A warp does a short one by
// itself, the whole CTA a long one.
constexpr int kShort = 16;
template <typename T, int ACCESS>
__global__ void __launch_bounds__(kThreads) join_kernel(int d, float scale, const __grid_constant__ Segments s, const __grid_constant__ Open open, T* __restrict__ out) {
  __shared__ __align__(16) float sums[kWarps][kGroup];
  __shared__ int64_t long_row[kWarps];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = blockIdx.y * kGroup + 4 * lane;
  const int64_t c0 = (int64_t)blockIdx.x * kWarps, c = c0 + warp;
  const int64_t row = c < s.stretches ? open.row[c] : -1;
  const auto key_of_tail = [&](int64_t q) { return s.key[(q + 1) * s.stretch - 1]; };
  const auto goes_on = [&](int64_t q, uint32_t key) { return q < s.stretches && s.key[q * s.stretch] == key; };
  const auto add = [&](f32x2 (&acc)[2], const float* from, int64_t q) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(from + q * open.width + blockIdx.y * kGroup + 4 * lane));
    acc[0] = plus2(acc[0], pair_of(v.x, v.y));
    acc[1] = plus2(acc[1], pair_of(v.z, v.w));
  };
  const auto write = [&](int64_t to, f32x2 (&acc)[2]) {
    acc[0] = mul2(acc[0], both(scale));
    acc[1] = mul2(acc[1], both(scale));
    Four<T, ACCESS> v;
    v.set(acc);
    v.store(out + to * d + col, d - col);
  };
  bool is_long = false;
  if (row >= 0) {
    // (the stretches of a segment lie side by side)
    const int count = __popc(__ballot_sync(0xffffffffu, goes_on(c + 1 + lane, key_of_tail(c))));
    is_long = count >= kShort;
    if (!is_long) {
      f32x2 acc[2] = {};
      add(acc, open.tail, c);
#pragma unroll
      for (int q = 0; q < kShort; ++q)
        if (q < count) add(acc, open.head, c + 1 + q);
      write(row, acc);
    }
  }
  if (lane == 0) long_row[warp] = is_long ? row : -1;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) {
    if (long_row[w] < 0) continue;  // for all threads alike
    const uint32_t key = key_of_tail(c0 + w);
    f32x2 acc[2] = {};
    if (warp == 0) add(acc, open.tail, c0 + w);
    int64_t q = c0 + w + 1 + warp;
    for (; goes_on(q + 3 * kWarps, key); q += 4 * kWarps) {  // (stretches of a segment lie side by side)
#pragma unroll
      for (int u = 0; u < 4; ++u) add(acc, open.head, q + u * kWarps);
    }
    for (; goes_on(q, key); q += kWarps) add(acc, open.head, q);
    *reinterpret_cast<ulonglong2*>(&sums[warp][4 * lane]) = make_ulonglong2(acc[0], acc[1]);
    __syncthreads();
    if (warp == 0) {
      f32x2 all[2] = {};
#pragma unroll
      for (int u = 0; u < kWarps; ++u) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sums[u][4 * lane]);
        all[0] = plus2(all[0], v.x);
        all[1] = plus2(all[1], v.y);
      }
      write(long_row[w], all);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- few places
constexpr int kOneLaunch = 1024, kFewWarps = kOneLaunch / 32, kShortSegment = 32;
constexpr unsigned long long kNobody = ~0ull;
constexpr int64_t kClearedBeside = 1 << 24;  // bytes of a table that this kernel clears itself

// Sorts a number of every thread of the CTA, in ascending order (a bitonic network): partners up to 16 lanes away by shuffles, the others by shared memory.
// `count` of them, from the first thread's on, are not the largest number there is.
template <int THREADS, typename N>
__device__ __forceinline__ N sort_block(N v, N* room, int count) {
  const int i = threadIdx.x;
#pragma unroll
  for (int size = 2; size <= THREADS; size *= 2) {
    if (size / 2 >= count) break;
#pragma unroll
    for (int apart = size / 2; apart > 0; apart /= 2) {
      N other;
      if (apart >= 32) {
        __syncthreads();
        room[i] = v;
        __syncthreads();
        other = room[i ^ apart];
      } else {
        other = __shfl_xor_sync(0xffffffffu, v, apart);
      }
      const bool lower = ((i & apart) == 0) == ((i & size) == 0);
      if ((v > other) == lower) v = other;
    }
  }
  return v;
}

// CTA x of gridDim.x has every gridDim.x-th segment, 128 columns of it, and every gridDim.x-th row that is to be zero (of the first `clear` rows of a whole table).
template <typename T, typename I, int ACCESS>
__global__ void __launch_bounds__(kOneLaunch, 1) few_kernel(const T* __restrict__ dy, int64_t ld, const I* __restrict__ ids, int m, uint32_t rows, int64_t clear, int d, float scale, T* __restrict__ out,
                                                            int64_t* __restrict__ looked_up, int64_t* __restrict__ count) {
  __shared__ __align__(16) unsigned long long room[kOneLaunch];
  __shared__ __align__(16) float sums[kFewWarps][kGroup];
  __shared__ uint32_t key_of_segment[kOneLaunch], place_of[kOneLaunch], before_warp[kFewWarps];
  __shared__ uint16_t start[kOneLaunch + 1];
  dependency_wait();
  release_dependents();
  const int i = threadIdx.x, lane = i & 31, warp = i >> 5, col = blockIdx.y * kGroup + 4 * lane, left = d - col;
  uint32_t key = i < m ? key_of(ids, i, rows) : rows;
  const unsigned long long sorted = sort_block<kOneLaunch>(key < rows ? (unsigned long long)key << 32 | (uint32_t)i : kNobody, room, m);
  __syncthreads();
  room[i] = sorted;
  __syncthreads();
  key = (uint32_t)(sorted >> 32);
  place_of[i] = (uint32_t)sorted;
  const bool there = sorted != kNobody, first = there && (i == 0 || (uint32_t)(room[i - 1] >> 32) != key);
  const uint32_t firsts = __ballot_sync(0xffffffffu, first);
  if (lane == 0) before_warp[warp] = __popc(firsts);
  __syncthreads();
  const uint32_t mine = before_warp[lane];  // (as many warps as lanes)
  const uint32_t number = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0u) + __popc(firsts & ((1u << lane) - 1u));
  if (first) {
    start[number] = (uint16_t)i;
    key_of_segment[number] = key;
  }
  const int kept = __syncthreads_count(there), segments = (int)__reduce_add_sync(0xffffffffu, mine);
  if (i == 0) start[segments] = (uint16_t)kept;
  __syncthreads();
  const auto add = [&](f32x2 (&acc)[2], int from, int to) {
    for (int p = from; p < to; p += kRowsAhead) {
      Four<T, ACCESS> v[kRowsAhead];
#pragma unroll
      for (int q = 0; q < kRowsAhead; ++q) v[q].load(dy + (int64_t)place_of[min(p + q, kOneLaunch - 1)] * ld + col, p + q < to ? left : 0);
#pragma unroll
      for (int q = 0; q < kRowsAhead; ++q) {
        f32x2 f[2];
        v[q].get(f);
        acc[0] = plus2(acc[0], f[0]);
        acc[1] = plus2(acc[1], f[1]);
      }
    }
  };
  const auto write = [&](int s, f32x2 (&acc)[2]) {
    acc[0] = mul2(acc[0], both(scale));
    acc[1] = mul2(acc[1], both(scale));
    Four<T, ACCESS> v;
    v.set(acc);
    v.store(out + (int64_t)(looked_up != nullptr ? (uint32_t)s : key_of_segment[s]) * d + col, left);
  };
  // short segments a warp each, long ones a 32nd of their places a warp
  for (int s = blockIdx.x + warp * gridDim.x; s < segments; s += kFewWarps * gridDim.x) {
    if (start[s + 1] - start[s] > kShortSegment) continue;
    f32x2 acc[2] = {};
    add(acc, start[s], start[s + 1]);
    write(s, acc);
  }
  for (int s = blockIdx.x; s < segments; s += gridDim.x) {
    const int from = start[s], places = start[s + 1] - from;
    if (places <= kShortSegment) continue;  // for all threads alike
    f32x2 acc[2] = {};
    add(acc, from + places * warp / kFewWarps, from + places * (warp + 1) / kFewWarps);
    *reinterpret_cast<ulonglong2*>(&sums[warp][4 * lane]) = make_ulonglong2(acc[0], acc[1]);
    __syncthreads();
    if (warp == 0) {
      acc[0] = acc[1] = 0ull;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sums[w][4 * lane]);
        acc[0] = plus2(acc[0], v.x);
        acc[1] = plus2(acc[1], v.y);
      }
      write(s, acc);
    }
    __syncthreads();
  }
  Four<T, ACCESS> zero;
  const f32x2 none[2] = {};
  zero.set(none);
  if (looked_up != nullptr) {
    for (int r = segments + blockIdx.x + warp * gridDim.x; r < m; r += kFewWarps * gridDim.x) zero.store(out + (int64_t)r * d + col, left);
    if (blockIdx.x == 0 && blockIdx.y == 0) {
      if (i < m) looked_up[i] = i < segments ? (int64_t)key_of_segment[i] : -1;
      if (i == 0) *count = segments;
    }
  } else {
    for (int64_t r = blockIdx.x + (int64_t)warp * gridDim.x; r < clear; r += (int64_t)kFewWarps * gridDim.x) {
      int low = 0, high = segments;  // the first segment whose row is not in front of this one
      while (low < high) {
        const int middle = (low + high) / 2;
        if (key_of_segment[middle] < (uint32_t)r) low = middle + 1;
        else high = middle;
      }
      if (low == segments || key_of_segment[low] != (uint32_t)r) zero.store(out + r * d + col, left);
    }
  }
}

// ---------------------------------------------------------------- few rows
// A CTA has `each` places, 128 columns of them: it sorts them by row while they come to shared memory, and leaves a sum for every row that is among them.
// (Places that need more than one CTA an SM: the sorting is not hidden any more, 236,000 of 1000 rows took 80 us and 68 with all of them sorted.  400 places are what float32
// rows leave room for, with some to spare; twice as many of 16-bit rows were not tried.  More rows
// times pieces of 128 columns: as many CTAs join them, 2000 x 128 of 2000 rows took 16 us and 10, of 1000 rows 11 and 10.)
constexpr int kLabels = 1024, kLabelThreads = 512, kLabelWarps = kLabelThreads / 32, kMostPlaces = 400, kLeastPlaces = 32;
constexpr uint16_t kNoSlot = 0xffffu;
static_assert(kLabels <= 1 << 22 && kMostPlaces < kLabelThreads, "a row and a place are one number of 32 bits, and none is the largest");
static_assert(kSmCount <= kLabelThreads, "a thread has a CTA's slot");

struct Labels {
  int64_t m, width;
  uint32_t rows;
  int d, each, ctas, slots;
  float* part;      // [ctas][slots][width]
  uint16_t* where;  // [rows][ctas]: a row's slot
  // only the rows that were looked up
  int words;
  uint32_t* seen;      // [words][ctas]: a bit for every row
  int64_t* looked_up;  // null: the whole table
  int64_t* count;
};

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(BYTES) : "memory");
}

template <typename T, typename I, int ACCESS>
__global__ void __launch_bounds__(kLabelThreads, 1) labels_kernel(const T* __restrict__ dy, int64_t ld, const I* __restrict__ ids, const __grid_constant__ Labels a) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ __align__(16) float sums[kLabelWarps][kGroup];
  __shared__ uint32_t room[kLabelThreads], before_warp[kLabelWarps], long_of[kLabelWarps];
  __shared__ uint16_t place_of[kLabelThreads], start[kLabelThreads + 1], slot[kLabels];
  T* const tile = reinterpret_cast<T*>(smem_raw);  // [each][128]
  dependency_wait();
  release_dependents();
  const int i = threadIdx.x, lane = i & 31, warp = i >> 5, col = blockIdx.y * kGroup + 4 * lane, left = a.d - col;
  const int64_t from = (int64_t)blockIdx.x * a.each;
  const int n = (int)min((int64_t)a.each, a.m - from);
  uint32_t key = i < n ? key_of(ids, from + i, a.rows) : a.rows;
  for (int p = warp; p < n; p += kLabelWarps) {
    const T* const at = dy + (from + p) * ld + col;
#pragma unroll
    for (int q = 0; q < Four<T, ACCESS>::kPieces; ++q) {
      constexpr int kEach = Four<T, ACCESS>::kEach;
      T* const to = tile + p * kGroup + 4 * lane + q * kEach;
      if (q * kEach >= left) continue;  // (what is there instead meets no column that exists)
      if constexpr (ACCESS >= 4) copy_async<ACCESS>(to, at + q * kEach);
      else *to = at[q];
    }
  }
  for (int r = i; r < (int)a.rows; r += kLabelThreads) slot[r] = kNoSlot;
  const uint32_t sorted = sort_block<kLabelThreads>(key < a.rows ? key << 9 | (uint32_t)i : ~0u, room, n);
  __syncthreads();
  room[i] = sorted;
  __syncthreads();
  key = sorted >> 9;
  place_of[i] = (uint16_t)(sorted & 511u);
  const bool there = sorted != ~0u, first = there && (i == 0 || room[i - 1] >> 9 != key);
  const uint32_t firsts = __ballot_sync(0xffffffffu, first);
  if (lane == 0) before_warp[warp] = __popc(firsts);
  __syncthreads();
  const uint32_t mine = lane < kLabelWarps ? before_warp[lane] : 0u;
  const uint32_t number = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0u) + __popc(firsts & ((1u << lane) - 1u));
  if (first) {
    start[number] = (uint16_t)i;
    slot[key] = (uint16_t)number;
  }
  const int kept = __syncthreads_count(there), segments = (int)__reduce_add_sync(0xffffffffu, mine);
  if (i == 0) start[segments] = (uint16_t)kept;
  __syncthreads();
  const uint32_t longs = __ballot_sync(0xffffffffu, i < segments && start[i + 1] - start[i] > kShortSegment);
  if (lane == 0) long_of[warp] = longs;
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  const auto add = [&](f32x2 (&acc)[2], int from, int to) {
#pragma unroll 4
    for (int p = from; p < to; ++p) {
      const Four<T, 4 * (int)sizeof(T)> v = *reinterpret_cast<const Four<T, 4 * (int)sizeof(T)>*>(tile + place_of[p] * kGroup + 4 * lane);
      f32x2 f[2];
      v.get(f);
      acc[0] = plus2(acc[0], f[0]);
      acc[1] = plus2(acc[1], f[1]);
    }
  };
  const auto write = [&](int s, const f32x2 (&acc)[2]) {
    *reinterpret_cast<ulonglong2*>(a.part + ((int64_t)blockIdx.x * a.slots + s) * a.width + blockIdx.y * kGroup + 4 * lane) = make_ulonglong2(acc[0], acc[1]);
  };
  // short segments a warp each, long ones a part of their places a warp
  for (int s = warp; s < segments; s += kLabelWarps) {
    if (start[s + 1] - start[s] > kShortSegment) continue;
    f32x2 acc[2] = {};
    add(acc, start[s], start[s + 1]);
    write(s, acc);
  }
  for (int word = 0; word < kLabelWarps; ++word)
    for (uint32_t bits = long_of[word]; bits != 0u; bits &= bits - 1u) {  // for all threads alike
      const int s = 32 * word + __ffs((int)bits) - 1, from = start[s], places = start[s + 1] - from;
      f32x2 acc[2] = {};
      add(acc, from + places * warp / kLabelWarps, from + places * (warp + 1) / kLabelWarps);
      *reinterpret_cast<ulonglong2*>(&sums[warp][4 * lane]) = make_ulonglong2(acc[0], acc[1]);
      __syncthreads();
      if (warp == 0) {
        acc[0] = acc[1] = 0ull;
#pragma unroll
        for (int w = 0; w < kLabelWarps; ++w) {
          const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sums[w][4 * lane]);
          acc[0] = plus2(acc[0], v.x);
          acc[1] = plus2(acc[1], v.y);
        }
        write(s, acc);
      }
      __syncthreads();
    }
  if (blockIdx.y != 0) return;
  for (int r = i; r < 32 * a.words; r += kLabelThreads) {
    const uint16_t s = r < (int)a.rows ? slot[r] : kNoSlot;
    if (r < (int)a.rows) a.where[(int64_t)r * a.ctas + blockIdx.x] = s;
    const uint32_t those = __ballot_sync(0xffffffffu, s != kNoSlot);
    if (lane == 0 && a.looked_up != nullptr) a.seen[(r >> 5) * a.ctas + blockIdx.x] = those;
  }
}

// A row's sums over the CTAs, in their order: a CTA to a row, 128 columns of it.  Where only the rows that were looked up are wanted (SOME) the CTAs behind those clear what
// is behind the last of them.
template <typename T, int ACCESS, bool SOME>
__global__ void __launch_bounds__(kLabelThreads, 2) label_rows_kernel(float scale, const __grid_constant__ Labels a, T* __restrict__ out) {
  __shared__ __align__(16) float sums[kLabelWarps][kGroup];
  __shared__ uint32_t list[kLabelThreads], before_warp[kLabelWarps], seen[SOME ? kLabels / 32 : 1];
  dependency_wait();
  release_dependents();
  const int i = threadIdx.x, lane = i & 31, warp = i >> 5, row = blockIdx.x, col = blockIdx.y * kGroup + 4 * lane;
  int64_t to = row;
  if constexpr (SOME) {
    const int needed = row < (int)a.rows ? (row >> 5) + 1 : a.words;
    for (int w = warp; w < needed; w += kLabelWarps) {
      uint32_t any = 0u;
      for (int c = lane; c < a.ctas; c += 32) any |= __ldg(a.seen + w * a.ctas + c);
      any = __reduce_or_sync(0xffffffffu, any);
      if (lane == 0) seen[w] = any;
    }
    __syncthreads();
    uint32_t before = 0u, all = 0u;
    for (int w = lane; w < needed; w += 32) {
      all += __popc(seen[w]);
      before += __popc(w < row >> 5 ? seen[w] : w == row >> 5 ? seen[w] & ((1u << (row & 31)) - 1u) : 0u);
    }
    to = __reduce_add_sync(0xffffffffu, before);
    all = __reduce_add_sync(0xffffffffu, all);
    if (row >= (int)a.rows) {
      Four<T, ACCESS> zero;
      const f32x2 none[2] = {};
      zero.set(none);
      const int cta = row - (int)a.rows, ctas = gridDim.x - (int)a.rows;
      for (int64_t r = (int64_t)all + cta * kLabelWarps + warp; r < a.m; r += ctas * kLabelWarps) {
        zero.store(out + r * a.d + col, a.d - col);
        if (lane == 0 && blockIdx.y == 0) a.looked_up[r] = -1;
      }
      if (cta == 0 && blockIdx.y == 0 && i == 0) *a.count = all;
      return;
    }
    if (((seen[row >> 5] >> (row & 31)) & 1u) == 0u) return;  // for all threads alike
    if (i == 0 && blockIdx.y == 0) a.looked_up[to] = row;
  }
  f32x2 acc[2] = {};
  const uint16_t slot = i < a.ctas ? __ldg(a.where + (int64_t)row * a.ctas + i) : kNoSlot;
  const uint32_t those = __ballot_sync(0xffffffffu, slot != kNoSlot);
  if (lane == 0) before_warp[warp] = __popc(those);
  __syncthreads();
  const uint32_t mine = lane < kLabelWarps ? before_warp[lane] : 0u, before = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0u);
  const int count = (int)__reduce_add_sync(0xffffffffu, mine);
  if (slot != kNoSlot) list[before + __popc(those & ((1u << lane) - 1u))] = (uint32_t)(i * a.slots + slot);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < (kSmCount + kLabelWarps - 1) / kLabelWarps; ++u) {
    const int q = warp + u * kLabelWarps;
    if (q >= count) continue;
    const float4 v = __ldg(reinterpret_cast<const float4*>(a.part + list[q] * a.width + blockIdx.y * kGroup + 4 * lane));
    acc[0] = plus2(acc[0], pair_of(v.x, v.y));
    acc[1] = plus2(acc[1], pair_of(v.z, v.w));
  }
  *reinterpret_cast<ulonglong2*>(&sums[warp][4 * lane]) = make_ulonglong2(acc[0], acc[1]);
  __syncthreads();
  if (warp != 0) return;
  acc[0] = acc[1] = 0ull;
#pragma unroll
  for (int w = 0; w < kLabelWarps; ++w) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sums[w][4 * lane]);
    acc[0] = plus2(acc[0], v.x);
    acc[1] = plus2(acc[1], v.y);
  }
  acc[0] = mul2(acc[0], both(scale));
  acc[1] = mul2(acc[1], both(scale));
  Four<T, ACCESS> v;
  v.set(acc);
  v.store(out + to * a.d + col, a.d - col);
}

// ---------------------------------------------------------------- host
template <typename T, typename I, int ACCESS>
static void lookup_as(const void* table, int64_t ld, int64_t rows, int64_t d, const void* ids, int64_t m, float scale, void* out, cudaStream_t st) {
  const int vectors = (int)(d * (int64_t)sizeof(T) / ACCESS);
  launch_dependent(lookup_kernel<T, I, ACCESS>, dim3((unsigned)ceil_div(m * vectors, kThreads * kAhead)), kThreads, 0, st, (const T*)table, ld, rows, vectors, (const I*)ids, m, scale,
                   (T*)out);
}
template <typename T, typename I>
static void lookup(const void* table, int64_t ld, int64_t rows, int64_t d, const void* ids, int64_t m, float scale, void* out, cudaStream_t st) {
  int access = 16;
  while (access > (int)sizeof(T) && (!aligned(table, access) || !aligned(out, access) || d * (int64_t)sizeof(T) % access != 0 || ld * (int64_t)sizeof(T) % access != 0)) access /= 2;
  if (access == 16) lookup_as<T, I, 16>(table, ld, rows, d, ids, m, scale, out, st);
  else if (access == 8) lookup_as<T, I, 8>(table, ld, rows, d, ids, m, scale, out, st);
  else if (access == 4 || sizeof(T) == 4) lookup_as<T, I, 4>(table, ld, rows, d, ids, m, scale, out, st);
  else if constexpr (sizeof(T) == 2) lookup_as<T, I, 2>(table, ld, rows, d, ids, m, scale, out, st);
}

// What a gradient needs of the workspace, in bytes from its start.
struct Plan {
  int64_t m, d;
  int stretch, tiles, bits, passes;
  int64_t stretches, width;
  int64_t key[2], place[2], counts[2], count_bytes, totals, in_tile, of_tile, head, tail, row, bytes;
};
static Plan plan(int64_t m, int64_t rows, int64_t d) {
  Plan p{};
  p.m = m;
  p.d = d;
  if (m <= kOneLaunch) return p;
  // Short stretches where there are few places: a stretch's rows are added one after the other.  Long ones where segments go over many of them: 236,000 places of
  // 172 rows took 69 us in stretches of 32 and 72 of 16, 121,000 of 2.4 M rows 84.7 and 79.6.
  p.stretch = m <= 16384 ? 8 : rows < m / 8 ? 32 : 16;
  p.tiles = (int)ceil_div(m, kTile);
  int bits = 1;
  while ((rows >> bits) != 0) ++bits;
  p.passes = m <= kFew ? 0 : (bits + kMaxBits - 1) / kMaxBits;
  p.bits = p.passes == 0 ? 0 : (bits + p.passes - 1) / p.passes;
  p.stretches = ceil_div(m, p.stretch);
  p.width = ceil_div(d, kGroup) * kGroup;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t from = at;
    at += ceil_div(bytes, 256) * 256;
    return from;
  };
  for (int b = 0; b < (p.passes > 1 ? 2 : 1); ++b) {
    p.key[b] = take(4 * m);
    p.place[b] = take(4 * m);
  }
  if (p.passes > 0) {
    p.count_bytes = ((int64_t)4 << p.bits) * p.tiles;
    for (int b = 0; b < (p.passes > 1 ? 2 : 1); ++b) p.counts[b] = take(p.count_bytes);
    p.totals = take((int64_t)4 << p.bits);
  }
  p.in_tile = take(4 * p.stretches);
  p.of_tile = take(4 * ((int64_t)p.tiles + 1));
  p.head = take(4 * p.stretches * p.width);
  p.tail = take(4 * p.stretches * p.width);
  p.row = take(8 * p.stretches);
  p.bytes = at;
  return p;
}

static Clear clear_of(void* at, int64_t bytes) {
  Clear c{(uint8_t*)at, 0, 0, 0};
  c.front = (16 - (int64_t)(reinterpret_cast<uintptr_t>(at) & 15)) & 15;
  if (c.front > bytes) c.front = bytes;
  c.whole = (bytes - c.front) / 16;
  c.behind = (bytes - c.front) % 16;
  return c;
}

// Sorts the places (and clears `bytes` bytes from `zero` on beside it); the pairs' final place.
template <typename I>
static Pairs sort(const Plan& p, const I* ids, uint32_t rows, char* ws, void* zero, int64_t bytes, cudaStream_t st) {
  Pairs pairs[2];
  for (int b = 0; b < 2; ++b) pairs[b] = Pairs{(uint32_t*)(ws + p.key[b]), (uint32_t*)(ws + p.place[b])};
  Clears clears{{clear_of(zero, bytes), clear_of(nullptr, 0)}};
  if (p.passes > 1) clears.of[1] = clear_of(ws + p.counts[1], p.count_bytes);
  const int64_t words = clears.of[0].whole + clears.of[1].whole;
  const int64_t wanted = words == 0 && bytes == 0 ? 0 : ceil_div(words + 1, kThreads * kClearEach);
  const unsigned more = (unsigned)(wanted < 8 * kSmCount ? wanted : 8 * kSmCount);
  if (p.passes == 0) {
    const int ctas = (int)ceil_div(p.m, 4 * kWarps);
    launch_dependent(rank_kernel<I>, dim3(ctas + more), kThreads, 0, st, ids, (int)p.m, rows, pairs[0], ctas, clears);
    return pairs[0];
  }
  uint32_t* const totals = (uint32_t*)(ws + p.totals);
  int to = p.passes & 1 ? 0 : 1;  // so that the last pass ends in pairs[0]
  for (int q = 0; q < p.passes; ++q, to ^= 1) {
    const Digit d{q * p.bits, p.bits}, next{(q + 1) * p.bits, p.bits};
    const Pairs in = pairs[to ^ 1], out = pairs[to];
    uint32_t *const counts = (uint32_t*)(ws + p.counts[q & 1]), *const counts_next = q + 1 < p.passes ? (uint32_t*)(ws + p.counts[(q + 1) & 1]) : nullptr;
    if (q == 0) launch_dependent(count_kernel<I>, dim3((unsigned)p.tiles + more), kThreads, 0, st, ids, p.m, rows, d, counts, p.tiles, clears);
    launch_dependent(tiles_kernel, dim3((unsigned)ceil_div((int64_t)1 << p.bits, 32)), 32 * kScanWarps, 0, st, counts, totals, p.tiles, 1 << p.bits);
    if (q == 0) launch_dependent(place_kernel<I, true>, dim3((unsigned)p.tiles), kThreads, 0, st, ids, in, p.m, rows, d, (const uint32_t*)counts, (const uint32_t*)totals, out, next, counts_next);
    else launch_dependent(place_kernel<I, false>, dim3((unsigned)p.tiles), kThreads, 0, st, ids, in, p.m, rows, d, (const uint32_t*)counts, (const uint32_t*)totals, out, next, counts_next);
    // (a third digit's counts go where the first one's were)
    if (q == 0 && p.passes > 2) (void)cudaMemsetAsync(counts, 0, (size_t)p.count_bytes, st);  // (what goes wrong is the last launch's error)
  }
  return pairs[0];
}

template <typename T, int ACCESS>
static void add_up(const Plan& p, const void* dy, int64_t ld, float scale, const Segments& s, const Open& open, void* out, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(p.stretches, kWarps), (unsigned)ceil_div(p.d, kGroup));
  launch_dependent(segment_kernel<T, ACCESS>, grid, kThreads, 0, st, (const T*)dy, ld, (int)p.d, scale, s, open, (T*)out);
  launch_dependent(join_kernel<T, ACCESS>, grid, kThreads, 0, st, (int)p.d, scale, s, open, (T*)out);
}

// CTAs of few_kernel: a warp to a segment at most, and enough to write a table of zeros.
template <typename T, int ACCESS>
static void add_few(const void* dy, int64_t ld, const void* ids, int index_dtype, int64_t m, bool clear, int64_t rows, int64_t d, float scale, void* out, int64_t* looked_up, int64_t* count, cudaStream_t st) {
  const int64_t slabs = ceil_div(d, kGroup), zeros = count == nullptr && clear ? rows : 0;
  int64_t ctas = std::max(ceil_div(m, kFewWarps), ceil_div(zeros, 16 * kFewWarps));
  ctas = std::min(ctas, std::max<int64_t>(1, kSmCount / slabs));
  const dim3 grid((unsigned)ctas, (unsigned)slabs);
  int64_t* const list = count != nullptr ? looked_up : nullptr;
  if (index_dtype == F2C_I64) launch_dependent(few_kernel<T, int64_t, ACCESS>, grid, kOneLaunch, 0, st, (const T*)dy, ld, (const int64_t*)ids, (int)m, (uint32_t)rows, zeros, (int)d, scale, (T*)out, list, count);
  else launch_dependent(few_kernel<T, int32_t, ACCESS>, grid, kOneLaunch, 0, st, (const T*)dy, ld, (const int32_t*)ids, (int)m, (uint32_t)rows, zeros, (int)d, scale, (T*)out, list, count);
}

// Few rows: how the places are dealt out, and the workspace.  `ctas` 0: not for these sizes.
static Labels labels(int64_t m, int64_t rows, int64_t d) {
  Labels a{};
  const int64_t slabs = ceil_div(d, kGroup);
  if (m <= kOneLaunch || rows == 0 || rows * slabs > kLabels || ceil_div(m, kMostPlaces) * slabs > kSmCount) return a;
  a.m = m;
  a.width = slabs * kGroup;
  a.rows = (uint32_t)rows;
  a.d = (int)d;
  a.each = (int)std::max<int64_t>(kLeastPlaces, ceil_div(m, kSmCount / slabs));
  a.ctas = (int)ceil_div(m, a.each);
  a.slots = (int)std::min<int64_t>(a.each, rows);
  a.words = (int)ceil_div(rows, 32);
  return a;
}
static int64_t label_parts(const Labels& a) { return ceil_div((int64_t)a.ctas * a.slots * a.width * 4, 256) * 256; }
static int64_t label_slots(const Labels& a) { return ceil_div((int64_t)a.ctas * a.rows * 2, 256) * 256; }
static int64_t label_bytes(const Labels& a) { return label_parts(a) + label_slots(a) + ceil_div((int64_t)a.ctas * a.words * 4, 256) * 256; }

template <typename T, int ACCESS>
static void add_labels(const char* op, const void* dy, int64_t ld, const void* ids, int index_dtype, const Labels& a, float scale, void* out, cudaStream_t st, int* rc) {
  const dim3 grid((unsigned)a.ctas, (unsigned)ceil_div(a.d, kGroup));
  const int bytes = a.each * kGroup * (int)sizeof(T);
  if (index_dtype == F2C_I64) {
    if ((*rc = allow_smem(op, (const void*)labels_kernel<T, int64_t, ACCESS>, kMostPlaces * kGroup * (int)sizeof(T)))) return;
    launch_dependent(labels_kernel<T, int64_t, ACCESS>, grid, kLabelThreads, bytes, st, (const T*)dy, ld, (const int64_t*)ids, a);
  } else {
    if ((*rc = allow_smem(op, (const void*)labels_kernel<T, int32_t, ACCESS>, kMostPlaces * kGroup * (int)sizeof(T)))) return;
    launch_dependent(labels_kernel<T, int32_t, ACCESS>, grid, kLabelThreads, bytes, st, (const T*)dy, ld, (const int32_t*)ids, a);
  }
  const unsigned more = a.looked_up == nullptr ? 0u : (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(a.m, 8 * kLabelWarps), 2 * kSmCount / grid.y));
  if (more == 0) launch_dependent(label_rows_kernel<T, ACCESS, false>, dim3(a.rows, grid.y), kLabelThreads, 0, st, scale, a, (T*)out);
  else launch_dependent(label_rows_kernel<T, ACCESS, true>, dim3(a.rows + more, grid.y), kLabelThreads, 0, st, scale, a, (T*)out);
}

static int check(const char* op, int dtype, int index_dtype, int64_t m, int64_t rows, int64_t d) {
  F2C_REQUIRE(is_float_dtype(dtype), F2C_ERR_UNSUPPORTED, "%s: rows must be float32, float16 or bfloat16", op);
  F2C_REQUIRE(is_index_dtype(index_dtype), F2C_ERR_UNSUPPORTED, "%s: ids must be int32 or int64", op);
  F2C_REQUIRE(m >= 0 && rows >= 0 && d >= 0, F2C_ERR_INVALID, "%s: negative size", op);
  F2C_REQUIRE(m <= kMaxPlaces && rows <= kMaxRows && d <= kMaxColumns && m * ceil_div(d, kGroup) <= 1ll << 33, F2C_ERR_LIMIT,
              "%s: more than 2^30 ids, 2^31 - 2 rows, 2^20 columns or 2^33 pieces of 128 columns", op);
  return F2C_OK;
}

}  // namespace emb
}  // namespace f2c

using namespace f2c;

extern "C" int f2c_embedding(const void* table, int64_t ld, int dtype, int64_t rows, int64_t d, const void* ids, int index_dtype, int64_t m, float scale, void* out, void* stream) {
  const char* op = "embedding";
  if (const int rc = emb::check(op, dtype, index_dtype, m, rows, d)) return rc;
  if (m == 0 || d == 0) return F2C_OK;
  F2C_REQUIRE((table || rows == 0) && ids && out, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(rows <= 1 || ld >= d, F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  cudaStream_t st = (cudaStream_t)stream;
  const bool wide = index_dtype == F2C_I64;
  if (dtype == F2C_F32) (wide ? emb::lookup<float, int64_t> : emb::lookup<float, int32_t>)(table, ld, rows, d, ids, m, scale, out, st);
  else if (dtype == F2C_F16) (wide ? emb::lookup<__half, int64_t> : emb::lookup<__half, int32_t>)(table, ld, rows, d, ids, m, scale, out, st);
  else (wide ? emb::lookup<__nv_bfloat16, int64_t> : emb::lookup<__nv_bfloat16, int32_t>)(table, ld, rows, d, ids, m, scale, out, st);
  return check_launch(op);
}

extern "C" int64_t f2c_embedding_backward_workspace(int64_t m, int64_t rows, int64_t d) {
  if (m <= 0 || rows < 0 || d <= 0 || m > emb::kMaxPlaces || rows > emb::kMaxRows || d > emb::kMaxColumns) return 0;
  const emb::Labels few = emb::labels(m, rows, d);
  return few.ctas > 0 ? emb::label_bytes(few) : emb::plan(m, rows, d).bytes;
}

extern "C" int f2c_embedding_backward(const void* dy, int64_t ldy, int dtype, const void* ids, int index_dtype, int64_t m, int64_t rows, int64_t d, float scale, void* grad,
                                      int64_t* looked_up, int64_t* count, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "embedding_backward";
  if (const int rc = emb::check(op, dtype, index_dtype, m, rows, d)) return rc;
  const bool dense = count == nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  F2C_REQUIRE(dense || looked_up || m == 0, F2C_ERR_INVALID, "%s: null pointer", op);
  if (dense && rows > 0 && d > 0) {
    F2C_REQUIRE(grad, F2C_ERR_INVALID, "%s: null pointer", op);
    F2C_REQUIRE(rows * d <= 1ll << 40, F2C_ERR_LIMIT, "%s: more than 2^40 values", op);
  }
  if (m > 0 && d > 0) {
    F2C_REQUIRE(dy && ids && (grad || (dense && rows == 0)), F2C_ERR_INVALID, "%s: null pointer", op);
    F2C_REQUIRE(m == 1 || ldy >= d, F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
    const int64_t need = f2c_embedding_backward_workspace(m, rows, d);
    F2C_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 256)), F2C_ERR_INVALID, "%s: the workspace must have %lld bytes, 256-byte aligned", op, (long long)need);
  }
  const int64_t bytes = dense ? rows * d * dtype_size(dtype) : 0;
  // (few places and a large table: cleared by itself.  The kernel's warps look every row up among the places': 2.4 M rows of 128 bytes took 364 us so, and 56 this way.)
  const bool cleared = bytes > 0 && (m == 0 || d == 0 || (m <= emb::kOneLaunch && bytes > emb::kClearedBeside));
  if (cleared) {
    const cudaError_t e = cudaMemsetAsync(grad, 0, (size_t)bytes, st);
    if (e != cudaSuccess) return set_error(F2C_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
  }
  if (!dense && (m == 0 || d == 0)) {
    cudaError_t e = cudaMemsetAsync(count, 0, 8, st);
    if (e == cudaSuccess && m > 0) e = cudaMemsetAsync(looked_up, 0xff, (size_t)m * 8, st);
    if (e != cudaSuccess) return set_error(F2C_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
  }
  if (m == 0 || d == 0 || (dense && rows == 0)) return F2C_OK;
  const int item = dtype_size(dtype), from = ckpt::access_of(dy, ldy, m, d, item), to = ckpt::access_of(grad, d, dense ? rows : m, d, item), access = from < to ? from : to;
  if (m <= emb::kOneLaunch) {
    F2C_BY_ROWS(emb::add_few, dtype, access, dy, ldy, ids, index_dtype, m, !cleared, rows, d, scale, grad, looked_up, count, st);
    return check_launch(op);
  }
  char* const ws = (char*)workspace;
  emb::Labels few = emb::labels(m, rows, d);
  if (few.ctas > 0) {
    few.part = (float*)ws;
    few.where = (uint16_t*)(ws + emb::label_parts(few));
    few.seen = (uint32_t*)(ws + emb::label_parts(few) + emb::label_slots(few));
    few.looked_up = dense ? nullptr : looked_up;
    few.count = count;
    int rc = F2C_OK;
    F2C_BY_ROWS(emb::add_labels, dtype, access, op, dy, ldy, ids, index_dtype, few, scale, grad, st, &rc);
    return rc != F2C_OK ? rc : check_launch(op);
  }
  const emb::Plan p = emb::plan(m, rows, d);
  const emb::Pairs sorted = index_dtype == F2C_I64 ? emb::sort(p, (const int64_t*)ids, (uint32_t)rows, ws, grad, bytes, st)
                                                       : emb::sort(p, (const int32_t*)ids, (uint32_t)rows, ws, grad, bytes, st);
  uint32_t *const in_tile = (uint32_t*)(ws + p.in_tile), *const of_tile = (uint32_t*)(ws + p.of_tile);
  const bool summed = !dense && p.tiles > emb::kTilesEach;
  if (!dense)
    launch_dependent(emb::number_kernel, dim3((unsigned)p.tiles), emb::kThreads, 0, st, (const uint32_t*)sorted.key, m, (uint32_t)rows, p.stretch, in_tile, of_tile, looked_up);
  if (summed) launch_dependent(emb::sum_kernel, dim3(1), emb::kSumThreads, 0, st, of_tile, p.tiles);
  const emb::Segments s{sorted.key, sorted.place, m, (uint32_t)rows, p.stretch, p.stretches, in_tile, of_tile, p.tiles, summed, dense ? nullptr : looked_up, count};
  const emb::Open open{(float*)(ws + p.head), (float*)(ws + p.tail), (int64_t*)(ws + p.row), p.width};
  F2C_BY_ROWS(emb::add_up, dtype, access, p, dy, ldy, scale, s, open, grad, st);
  return check_launch(op);
}
