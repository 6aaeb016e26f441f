// Newton-Schulz steps on stacks of matrices (f2c_orthogonalize) and the optimiser step around them (f2c_muon_step):
//   X = G / (|G|_F + eps);   A = X X^T,  R = b A + c A^2,  X <- a X + R X   for every step.
//
// What bounds it: the tensor cores where matrices are large (4096 x 4096 bfloat16: 1.32 ms for five steps, products of 1.3 PFLOP/s; 2048 x 2048 and
// 2048 x 8192 float32, three products for one: 2.3 to 2.4 ms), and the latency of 17 launches where they are not (1031 x 602 float32: 181 us).
//
// Products.  Three per step, on the 5th-generation tensor cores, one launch each (product_kernel).  A tile of a product has 128 rows (the
// lanes of TMEM) and up to 256 columns.  A and A^2 are symmetric: tiles wholly below the diagonal are left out, what lies on or above it is written
// twice.  Nothing is transposed in memory: an operand whose rows run along M or N instead of K is one that the MMA takes as it is, so a
// matrix of more rows than columns, which is worked on transposed, is read the other way round.  The sums' factors, b A, a X and - in the
// last step - the optimiser's update are the epilogue's.
//
// Precision.  Operands are half precision times a power of two for each matrix and step, chosen by a bound on the matrix' norm so that
// the smallest values keep their bits and the largest have room: X and A stay below 2^11, R below 60 * 2^10 for any coefficients that are
// accepted (infinity is 2^16; of the default ones R stays below 2.9 * 2^10).  Sums are single precision, the norm's double.
//  * bfloat16.  The first X is exact, A and R are rounded to 11 bits (R multiplies from the left: its rounding turns the singular
//    vectors by 2^-12 of R's size), or pairs where they have no more than 256 rows (the fewer, the less do roundings cancel out: 43 x 42 in bfloat16
//    3.0e-3 off without, of which the result's own rounding is 1.7e-3).  X's own rounding is noise of full rank, which the following steps multiply by up to the product of their
//    factors a, 3.4445^4 = 140 after the first, while large singular values only go to one: where that product is over 16, X is a pair of
//    half precision numbers (22 bits) and R X two products.  For matrices of rank 8 the result is 2.6e-3 off then, and 2.6e-2 without.
//  * float32, and float16, whose own 11 bits the result has to keep.  All operands are pairs, a product is three (high by high, high by low, low by high): 22 bits throughout.  The tensor
//    cores cut sums off instead of rounding them, for every 16 elements of K.  So the sums are taken out every 64 or 128 elements and added up in
//    registers, the small products are in front of the large one, and a X is not in the sum.  (Rank 3, 400 x 600: 2.5e-4 off without any of this,
//    2e-4 without the taking out.)
#include <math.h>

#include <algorithm>
#include <vector>

#include "newton_schulz.cuh"

namespace f2c {
namespace ns {

constexpr int kMaxParts = 1024, kLoadThreads = 256;  // parts of a matrix' norm
constexpr int kFirstEpilogueWarp = 4, kEpilogueWarps = 8, kThreads = 32 * (kFirstEpilogueWarp + kEpilogueWarps);  // warp 0: TMA, warp 1: MMA
constexpr int kM = 128, kK = 64, kMaxSums = 128, kMaxStages = 8;
constexpr size_t kRoom = kSmemLimit - 1024;  // dynamic shared memory

// Momentum, and the squares' sums of gridDim.x parts of every matrix.
template <typename T, int V>
__global__ void __launch_bounds__(kLoadThreads) norm_kernel(const __grid_constant__ Matrices s, double* parts) {
  dependency_wait();
  release_dependents();
  const int z = blockIdx.y;
  double sum = 0.0;
  for (int64_t i = ((int64_t)blockIdx.x * kLoadThreads + threadIdx.x) * V; i < s.size; i += (int64_t)gridDim.x * kLoadThreads * V) {
    float u[V];
    direction<T, V, true>(s, z, i, u);
#pragma unroll
    for (int e = 0; e < V; ++e) sum = fma((double)u[e], (double)u[e], sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __shared__ double sums[kLoadThreads / 32];
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kLoadThreads / 32; ++w) sum += sums[w];
    parts[z * kMaxParts + blockIdx.x] = sum;
  }
}

// X as half precision (and what that leaves, where `low` is given), and the steps' factors.
template <typename T, int V>
__global__ void __launch_bounds__(kLoadThreads) planes_kernel(const __grid_constant__ Matrices s, const __grid_constant__ Steps st, const double* parts,
                                                              __half* high, __half* low, int64_t rows, int64_t cols, int64_t ld, Factors* table) {
  dependency_wait();
  release_dependents();
  const int z = blockIdx.y;
  __shared__ double norm_s;
  if (threadIdx.x < 32) {
    double sum = 0.0;
    for (int q = threadIdx.x; q < gridDim.x; q += 32) sum += parts[z * kMaxParts + q];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x == 0) norm_s = sqrt(sum);
  }
  __syncthreads();
  const double norm = norm_s;
  const bool finite = norm <= 1e300;
  const int up = scale_up(norm);
  // u 2^up in two factors: the power itself may be out of range.  A matrix that is not finite becomes NaN.
  const float by = power2(up / 2), more = finite ? power2(up - up / 2) : __int_as_float(0x7fffffff);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    make_factors(st, norm, up, table + z * F2C_MAX_NS_STEPS);
  }
  __half* const hi = high + z * rows * ld;
  __half* const lo = low + z * rows * ld;
  for (int64_t i = ((int64_t)blockIdx.x * kLoadThreads + threadIdx.x) * V; i < s.size; i += (int64_t)gridDim.x * kLoadThreads * V) {
    float u[V];
    direction<T, V, false>(s, z, i, u);
    const int64_t at = ld == cols ? i : i / cols * ld + i % cols;
    Chunk<__half, V> h, l;
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const float v = u[q] * by * more;
      h.v[q] = __float2half_rn(v);
      l.v[q] = __float2half_rn(v - __half2float(h.v[q]));
    }
    *reinterpret_cast<Chunk<__half, V>*>(hi + at) = h;
    if (low != nullptr) *reinterpret_cast<Chunk<__half, V>*>(lo + at) = l;
  }
}

// No steps: X itself is the result.
template <typename T>
__global__ void __launch_bounds__(kLoadThreads) store_kernel(const __grid_constant__ Matrices s, const __half* high, const __half* low, int64_t rows, int64_t cols,
                                                             int64_t ld, const Factors* table) {
  dependency_wait();
  release_dependents();
  const int z = blockIdx.y;
  const float kappa = table[z * F2C_MAX_NS_STEPS].apply;
  for (int64_t i = (int64_t)blockIdx.x * kLoadThreads + threadIdx.x; i < s.size; i += (int64_t)gridDim.x * kLoadThreads) {
    const int64_t at = z * rows * ld + i / cols * ld + i % cols;
    const float x = kappa * (__half2float(high[at]) + (low != nullptr ? __half2float(low[at]) : 0.0f));
    T* const out = s.template result<T>(z) + i;
    *out = from_float<T>(s.listed ? s.keep * to_float(*out) - s.gain(rows, cols) * x : x);
  }
}

// ---------------------------------------------------------------- products
enum Mode { kGram, kPoly, kApply, kFinal };

struct Operand {
  int rows;     // of a CTA's part of a tile
  int turned;   // its rows run along K
  int planes;   // 1 or 2
  __host__ __device__ int bytes(int chunks) const { return rows * kK * 2 * chunks; }
};

struct Params {
  Operand a, b;
  int m, n, steps;                 // M, N of the product; steps of K
  int col_tiles, items;            // of one matrix
  int batch, stages;
  int chunks;                      // of 64 elements of K in a stage (of which there are `steps`)
  int split, parts_at;             // CTAs that take parts of K, and where in shared memory they put their sums together
  int symmetric;
  const Factors* factors;          // of this step
  const __half *add_high, *add_low;  // kPoly: As; kApply, kFinal: Xs
  __half *high, *low;              // result [n][m] (kGram and kPoly: symmetric); low null: none; ld and stack also Xs'
  int64_t ld, stack;               // elements between rows, and between matrices
  float gain;                      // kFinal, optimiser: times the result
  int issued;                      // tiles that are loaded and multiplied: all, or none (then the waits for their sums run out)
  int* error;
};

struct Bars {
  uint64_t full[kMaxStages], empty[kMaxStages], drain, acc_full[2], acc_empty[2];
  uint32_t tmem;
  int failed, lost;  // lost: of any CTA of the cluster
};

struct Maps { CUtensorMap a[2], b[2]; };  // high, low

struct Tile { int z, row, col; };
// Tile `item` of the list.  Symmetric products: row tile i starts with the column tile that its diagonal is in.
__device__ __forceinline__ Tile tile_of(const Params& p, int item) {
  Tile t;
  t.z = item / p.items;
  int i = item % p.items;
  if (!p.symmetric) {
    t.row = i / p.col_tiles;
    t.col = i % p.col_tiles;
    return t;
  }
  t.row = 0;
  for (int first = 0;; first = t.row * kM / p.b.rows) {  // (rows and columns of a tile have the same factor, ctas)
    if (i < p.col_tiles - first) {
      t.col = first + i;
      return t;
    }
    i -= p.col_tiles - first;
    ++t.row;
  }
}

// 32 values at `ld` from one another, as many as there are: all on the way before the first is used
template <typename T>
__device__ __forceinline__ void gather(const T* from, int64_t ld, int count, float (&v)[32]) {
  T raw[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) raw[j] = from[min(j, count - 1) * ld];
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = to_float(raw[j]);
}

template <typename T>
__device__ __forceinline__ void scatter(T* to, int64_t ld, int count, bool mine, const T (&v)[32]) {
  if (__all_sync(0xffffffffu, mine) && count == 32) {
#pragma unroll
    for (int j = 0; j < 32; ++j) to[j * ld] = v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (mine && j < count) to[j * ld] = v[j];
  }
}

// A lane's row of the product, 32 values from column `col` on (which exists), to where they belong; called by whole warps, whose rows start
// at `row0`.  A warp reads and writes 32 neighbours at a time: [column][row].  Symmetric, where half of the tiles are
// made: also [row][column] of what lies above the diagonal; a chunk with the diagonal has both sides.
template <int MODE, typename T>
__device__ __forceinline__ void store_values(const Params& p, const Matrices& s, const Factors& f, int z, int row0, int col, const uint32_t (&r)[32], bool lost) {
  const int row = row0 + (threadIdx.x & 31), count = min(32, p.n - col);
  const bool mine = row < p.m;
  const int64_t stack = z * p.stack, at = stack + (int64_t)col * p.ld + min(row, p.m - 1);
  const float by = lost ? __int_as_float(0x7fffffff) : MODE == kGram ? f.gram : MODE == kPoly ? f.poly_c : f.apply;
  float v[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]) * by;
  if constexpr (MODE != kGram) {
    const float other = MODE == kPoly ? f.poly_b : f.own;
    float more[32];
    gather(p.add_high + at, p.ld, count, more);
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = fmaf(other, more[j], v[j]);
    if (p.add_low != nullptr) {
      gather(p.add_low + at, p.ld, count, more);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = fmaf(other, more[j], v[j]);
    }
  }
  if constexpr (MODE == kFinal) {
    T* const out = s.template result<T>(z) + (int64_t)col * p.m + min(row, p.m - 1);
    T o[32];
    if (s.listed) {
      float w[32];
      gather(out, (int64_t)p.m, count, w);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = s.keep * w[j] - p.gain * v[j];
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) o[j] = from_float<T>(v[j]);
    scatter(out, (int64_t)p.m, count, mine, o);
  } else {
    union Half { __half h[32]; __half2 p[16]; uint4 v[4]; __device__ Half() {} };
    const int64_t across = stack + (int64_t)row * p.ld + col;
    const bool above = p.symmetric && col > row0 && mine;
    // One copy of the code for both planes: a short launch waits for its instructions to come from memory (1031 x 602 float32: 184 us, 205 with
    // two; 1500 x 1500 bfloat16: 224 and 243; long ones 1% the other way).  The reading in one copy keeps fewer loads on the way (12 x 1024 x 1024
    // bfloat16: 516 us, 437 so).
#pragma unroll 1
    for (__half* to = p.high; to != nullptr; to = to == p.high ? p.low : nullptr) {
      Half half;
#pragma unroll
      for (int j = 0; j < 16; ++j) half.p[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
      scatter(to + at, p.ld, count, mine, half.h);
      if (above) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (8 * q < count) *reinterpret_cast<uint4*>(to + across + 8 * q) = half.v[q];
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] -= __half2float(half.h[j]);  // what the low plane has to hold
    }
  }
}

__device__ __forceinline__ void add(uint32_t (&sum)[32], const uint32_t (&r)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j) sum[j] = __float_as_uint(__uint_as_float(sum[j]) + __uint_as_float(r[j]));
}

// CTAS 2: the two CTAs of a cluster work on 256 rows, each with 128 of them and half of the columns' operand in its shared memory; the
// first one issues the MMAs for both.  SPLIT: the CTAs of a cluster each take a part of K, put their sums together over distributed shared
// memory, and each has some of the columns' results to write (a kernel of its own: with both ways in one the registers spilled, 1.2 us a launch).
template <int MODE, typename T, int CTAS, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p, const __grid_constant__ Matrices s) {
  constexpr bool kWide = is_wide<T>;  // pairs by pairs: see above
  extern __shared__ unsigned char smem_raw[];
  __shared__ Bars bars;
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  const int split = SPLIT ? p.split : 1, group = CTAS * split, member = (int)blockIdx.x % group;
  const int rank = SPLIT ? 0 : member, part = SPLIT ? member : 0, first = (int)blockIdx.x / group, stride = (int)gridDim.x / group;
  const int step0 = p.steps * part / split, steps = p.steps * (part + 1) / split - step0;
  const int total = p.items * p.batch;
  const uint32_t a_bytes = (uint32_t)p.a.bytes(p.chunks), b_bytes = (uint32_t)p.b.bytes(p.chunks);  // of a plane of a stage
  const uint32_t b_at = a_bytes * p.a.planes, stage_bytes = b_at + b_bytes * p.b.planes;
  const int columns = p.b.rows * CTAS;  // of a tile
  const uint32_t tmem_columns = (uint32_t)columns * 2;  // two accumulators
  uint32_t left = kWaitLimit;  // (a constant: with a parameter in its place 4096 x 4096 bfloat16 took 1595 us instead of 1510)

  if (wid == 1) {
    if (CTAS == 2) alloc_tmem_pair(&bars.tmem, tmem_columns);
    else alloc_tmem(&bars.tmem, tmem_columns);
  }
  if (tid == 0) {
    for (int q = 0; q < p.stages; ++q) { init_bar(bars.full + q, 1); init_bar(bars.empty + q, 1); }
    init_bar(&bars.drain, 1);
    for (int b = 0; b < 2; ++b) { init_bar(bars.acc_full + b, 1); init_bar(bars.acc_empty + b, kEpilogueWarps * CTAS); }
    fence_bars();
    bars.failed = 0;
    bars.lost = 0;
  }
  fence_before();
  __syncthreads();
  if (group > 1) cluster_barrier();  // the other ones' barriers and shared memory are there
  fence_after();
  const uint32_t tmem = bars.tmem;
  int slot = 0;
  uint32_t round = 0;

  if (wid < kFirstEpilogueWarp) {
    const bool mine = elected() != 0u;
    if (wid != 1) {
      // ================= loads: a warp of its own for each operand, and one for their low planes
      if (mine) {
        prefetch_map(&maps.a[wid == 3]);
        prefetch_map(&maps.b[wid == 3]);
      }
      __syncwarp();
      dependency_wait();
      if (wid == 0) release_dependents();
      const bool high = wid != 3, of_a = high ? wid == 0 : p.a.planes > 1, of_b = high ? wid == 2 : p.b.planes > 1;
      const uint32_t smem0 = smem_u32(smem), a_at = high ? 0u : a_bytes, b_from = b_at + (high ? 0u : b_bytes);
      const uint32_t bars0 = CTAS == 2 ? peer_address(smem_u32(bars.full), 0) : smem_u32(bars.full);
      const int depth = p.chunks * kK;
      const auto load = [&](bool go, const Operand& o, const CUtensorMap* map, uint32_t dst, uint32_t bar, int k, int at, int z) {
        const int boxes = o.turned ? o.rows / 64 : p.chunks, box_bytes = o.turned ? depth * 128 : o.rows * 128;
        int x = o.turned ? at : k;
        const int y = o.turned ? k : at;
        for (int c = 0; c < boxes; ++c, x += 64, dst += (uint32_t)box_bytes) {
          if (CTAS == 2) tma_load_pair(go, map, dst, bar, x, y, z);
          else tma_load(go, map, dst, bar, x, y, z);
        }
      };
      const CUtensorMap *a_map = high ? &maps.a[0] : &maps.a[1], *b_map = high ? &maps.b[0] : &maps.b[1];
      for (int item = of_a || of_b ? first : p.issued; item < p.issued; item += stride) {
        const Tile t = tile_of(p, item);
        const int a_row = (t.row * CTAS + rank) * kM, b_row = t.col * columns + rank * p.b.rows;
        for (int i = 0; i < steps; ++i) {
          if (round > 0) wait_bar(bars.empty + slot, (round - 1) & 1, left);
          const bool go = mine && left != 0u;
          const uint32_t stage = smem0 + (uint32_t)slot * stage_bytes, bar = bars0 + (uint32_t)slot * 8u;
          expect_if(go && wid == 0 && rank == 0, bars.full + slot, stage_bytes * CTAS);
          if (of_a) load(go, p.a, a_map, stage + a_at, bar, (step0 + i) * depth, a_row, t.z);
          if (of_b) load(go, p.b, b_map, stage + b_from, bar, (step0 + i) * depth, b_row, t.z);
          if (++slot == p.stages) { slot = 0; ++round; }
        }
      }
    } else if (rank == 0) {
      // ================= MMAs
      const uint32_t idesc = instruction(kSumF32, kFormatF16, kM * CTAS, (uint32_t)columns) | (p.a.turned ? kTurnedA : 0u) | (p.b.turned ? kTurnedB : 0u);
      const auto done = [&](bool go, const uint64_t* bar) {
        if (CTAS == 2) commit_pair(go, bar);
        else commit(go, bar);
      };
      const uint32_t low = desc_low(smem_u32(smem), 0), a_low = low | desc_low(0, p.a.turned ? p.chunks * kK * 128 : kChunkAlongK);
      const uint32_t b_low = (low | desc_low(0, p.b.turned ? p.chunks * kK * 128 : kChunkAlongK)) + (b_at >> 4);
      const uint32_t a_step = p.a.turned ? kStepTurned : kStepAlongK, b_step = p.b.turned ? kStepTurned : kStepAlongK;
      const uint32_t a_chunk = p.a.turned ? 4 * kStepTurned : (uint32_t)p.a.rows * 8u, b_chunk = p.b.turned ? 4 * kStepTurned : (uint32_t)p.b.rows * 8u;
      // The products of a stage: the small ones first (what is cut off their sums is as small as they are), then the large one.
      const uint32_t a_small = a_bytes >> 4, b_small = b_bytes >> 4;
      const int products = p.a.planes + p.b.planes - 1;
      // Waits for a step are made behind the MMAs and commits of the one before, some of which the tensor cores still have to do meanwhile.
      const int mine_items = p.issued > first ? (p.issued - first + stride - 1) / stride : 0, all = mine_items * steps;
      uint32_t n = 0;  // accumulations begun: one a tile, or (pairs) one a step
      int done_steps = 0, i = 0;
      const auto wait_full = [&]() { wait_bar(bars.full + slot, round & 1, left); };
      const auto wait_acc = [&]() {  // of accumulation n
        if (n >= 2) wait_bar(bars.acc_empty + (n & 1u), ((n >> 1) - 1) & 1, left);
      };
      if (all > 0) wait_full();
      for (; done_steps < all; ++done_steps) {
        const bool fresh = kWide || i == 0, last = kWide || i + 1 == steps, more_steps = done_steps + 1 < all;
        if (++i == steps) i = 0;
        fence_after();
        const bool go = mine && left != 0u;
        const uint32_t at = (uint32_t)slot * (stage_bytes >> 4), acc = tmem + (n & 1u) * (uint32_t)columns;
        const uint64_t *const empty = bars.empty + slot, *const full_acc = bars.acc_full + (n & 1u);
        if (++slot == p.stages) { slot = 0; ++round; }
        if (last) ++n;
        bool more = !fresh;
        for (int q = 0; q < products; ++q) {
          const bool large = q + 1 == products, of_a = !large && q == 0 && p.a.planes > 1;  // the small product with A's low plane, or B's
          uint32_t a = a_low + at + (of_a ? a_small : 0u), b = b_low + at + (large || of_a ? 0u : b_small);
          for (int c = 0; c < p.chunks; ++c, a += a_chunk, b += b_chunk) {
#pragma unroll
            for (uint32_t e = 0; e < kK / 16; ++e) {
              if (CTAS == 2) mma_f16_pair(go, acc, desc(a + e * a_step), desc(b + e * b_step), idesc, more || e != 0);
              else mma_f16(go, acc, desc(a + e * a_step), desc(b + e * b_step), idesc, more || e != 0);
            }
            more = true;
            if (products > 1 && q == 0 && c == 0 && more_steps && last) wait_acc();
          }
        }
        done(go, empty);
        if (last) done(go, full_acc);
        if (products == 1 && more_steps && last) wait_acc();
        if (more_steps) wait_full();
      }
    }
  } else {
    // ================= epilogue: a warp has the TMEM lanes of its quarter and half of the columns, thread = row
    const int quarter = wid & 3, half = (wid - kFirstEpilogueWarp) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const auto leave = [&](uint32_t buf) {  // the accumulator has been read
      fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CTAS == 2) peer_arrive(peer_address(smem_u32(bars.acc_empty + buf), 0));
        else arrive(bars.acc_empty + buf);
      }
    };
    // In parts of K: 32 columns of sums to the CTA whose they are, there [this CTA][column][row]
    const auto tell = [&](int c0, const uint32_t (&r)[32]) {
      const int share = columns / split, owner = c0 / share;
      const uint32_t to = peer_address(smem_u32(smem) + (uint32_t)p.parts_at + 4u * (uint32_t)((part * share + c0 - owner * share) * kM + quarter * 32 + lane), (uint32_t)owner);
#pragma unroll
      for (int j = 0; j < 32; ++j) peer_store(to + (uint32_t)(j * kM) * 4u, r[j]);
    };
    const auto tell_lost = [&](bool lost) {
      if (lost && lane < split) peer_store(peer_address(smem_u32(&bars.lost), (uint32_t)lane), 1u);
    };
    uint32_t n = 0;
    dependency_wait();
    for (int item = first; item < total; item += stride) {
      const Tile at = tile_of(p, item);
      const int row0 = (at.row * CTAS + rank) * kM + quarter * 32, col0 = at.col * columns;
      const Factors f = p.factors[at.z * F2C_MAX_NS_STEPS];
      if constexpr (kWide) {
        // the sums of the steps are added up here, where additions round
        uint32_t sum[2][32] = {};
        const int width = columns / 2, mine = half * width;
        for (int i = 0; i < steps; ++i, ++n) {
          const uint32_t turn = n >> 1, buf = n & 1u;
          wait_bar(bars.acc_full + buf, turn & 1, left);
          __syncwarp();
          fence_after();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (c * 32 >= width) break;
            uint32_t r[32];
            tmem_ld32(lanes + buf * (uint32_t)columns + (uint32_t)(mine + c * 32), r);
            tmem_wait(r);
            add(sum[c], r);
          }
          leave(buf);
        }
        const bool lost = __any_sync(0xffffffffu, left == 0u);
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          const int col = col0 + mine + c * 32;
          if (c * 32 < width && col < p.n && !(p.symmetric && col + 31 < row0)) {  // (not wholly below the diagonal)
            if constexpr (SPLIT) tell(mine + c * 32, sum[0]);
            else store_values<MODE, T>(p, s, f, at.z, row0, col, sum[0], lost);
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) sum[0][j] = sum[1][j];
        }
        if constexpr (SPLIT) tell_lost(lost);
        __syncwarp();
      } else {
        const uint32_t turn = n >> 1, buf = n & 1u;
        const int cols = min(columns, p.n - col0);
        wait_bar(bars.acc_full + buf, turn & 1, left);
        const bool lost = __any_sync(0xffffffffu, left == 0u);
        fence_after();
        for (int c0 = half * 32; c0 < cols; c0 += 64) {
          if (p.symmetric && col0 + c0 + 31 < row0) continue;
          uint32_t r[32];
          tmem_ld32(lanes + buf * (uint32_t)columns + (uint32_t)c0, r);
          tmem_wait(r);
          if constexpr (SPLIT) tell(c0, r);
          else store_values<MODE, T>(p, s, f, at.z, row0, col0 + c0, r, lost);
          __syncwarp();
        }
        if constexpr (SPLIT) tell_lost(lost);
        leave(buf);
        ++n;
      }
    }
  }
  if (left == 0u) bars.failed = 1;
  __syncwarp();
  if constexpr (SPLIT) {
    // a cluster has one tile, whose columns its CTAs share: all sums have been told when all have got here, and are added in the order of K
    cluster_barrier();
    if (wid >= kFirstEpilogueWarp) {
      const int quarter = wid & 3, half = (wid - kFirstEpilogueWarp) >> 2, share = columns / split;
      const Tile at = tile_of(p, first);
      const int row0 = at.row * kM + quarter * 32;
      const Factors f = p.factors[at.z * F2C_MAX_NS_STEPS];
      const bool lost = bars.lost != 0;
      const float* told = reinterpret_cast<const float*>(smem + p.parts_at) + quarter * 32 + lane;
      for (int c0 = half * 32; c0 < share; c0 += 64) {
        const int col = at.col * columns + part * share + c0;
        if (col >= p.n) continue;
        uint32_t sum[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) sum[j] = __float_as_uint(told[(c0 + j) * kM]);
        for (int q = 1; q < split; ++q) {
          uint32_t more[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) more[j] = __float_as_uint(told[(q * share + c0 + j) * kM]);
          add(sum, more);
        }
        store_values<MODE, T>(p, s, f, at.z, row0, col, sum, lost);
      }
    }
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  if (bars.failed && rank == 0) {
    // copies in flight write to shared memory, MMAs in flight read it and write TMEM, of both CTAs: wait (bounded) for what was issued
    left = kWaitLimit;
    if (wid == 0) {
      for (int q = 0; q < p.stages; ++q) {
        const uint32_t uses = round + (q < slot ? 1u : 0u);
        if (uses > 0) wait_bar(bars.full + q, (uses - 1) & 1, left);
      }
    } else if (wid == 1) {
      const bool mine = elected() != 0u;  // who issued them
      if (CTAS == 2) commit_pair(mine, &bars.drain, 1);
      else commit(mine, &bars.drain);
      wait_bar(&bars.drain, 0, left);
    }
    __syncthreads();
  }
  if (CTAS == 2) cluster_barrier();
  if (wid == 1) {
    fence_after();
    if (CTAS == 2) free_tmem_pair(tmem, tmem_columns);
    else free_tmem(tmem, tmem_columns);
  }
  if (tid == 0 && bars.failed) report_wait(p.error, 5);
}

// ---------------------------------------------------------------- host
static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

struct Shape {
  int64_t batch, rows, cols;
  int64_t p() const { return rows < cols ? rows : cols; }
  int64_t ldx() const { return (cols + 7) / 8 * 8; }
  int64_t ldp() const { return (p() + 7) / 8 * 8; }
  int64_t x_bytes() const { return round256(2 * batch * rows * ldx()); }
  bool fine(bool wide) const { return wide || p() <= 256; }  // A and R are pairs
  int64_t p_bytes() const { return round256(2 * batch * p() * ldp()); }
};

// Planes of X in front of a step: 2 where all operands are pairs; otherwise see above (`exact`: the first X is).
static int x_planes(const Steps& st, int t, bool wide, bool exact) {
  if (wide) return 2;
  if (t == 0 && exact) return 1;
  double gain = 1.0;
  for (int q = t; q < st.count; ++q) {
    const double a = fabs((double)st.co[3 * q]);
    gain *= a > 1.0 ? a : 1.0;
  }
  return gain > 16.0 ? 2 : 1;
}

static int64_t workspace(const Shape& s, bool wide) {
  return 4 * s.x_bytes() + (s.fine(wide) ? 4 : 2) * s.p_bytes() + round256(8 * s.batch * kMaxParts) + round256((int64_t)sizeof(Factors) * F2C_MAX_NS_STEPS * s.batch);
}

struct Planes {
  __half *high, *low;
};

// Tiles of one matrix' product.
static int64_t tiles(int64_t m, int64_t n, int rows, int columns, bool symmetric) {
  const int64_t rt = ceil_div(m, rows), ct = ceil_div(n, columns);
  if (!symmetric) return rt * ct;
  int64_t items = 0;
  for (int64_t i = 0; i < rt; ++i) items += ct - i * rows / columns;
  return items;
}

// Pieces of 64 elements of K in a stage.  Pairs, whose sums are taken out after every stage: two (2048 x 8192 float32: 2.59 ms a step, 2.81 with one), but
// one of matrices of up to 1024 rows or columns, whose products are short anyway: the cutting off makes sums smaller, all alike, and
// the fewer singular values there are, the more it counts (1500 x 300: 3.3e-6 off with two).  bfloat16: one (4096 x 4096: 1.36 ms, 1.49 with two,
// of which fewer stages fit).
static int chunks_of(bool wide, int64_t p) { return wide && p > 1024 ? 2 : 1; }

struct Tiling { int ctas, columns, split; };

// The tiles of least cycles: rounds over the SMs of a tile's stages, which take the longer of their MMAs (half a cycle a column, 46 cycles at least,
// and 250 for the waits) and their bytes at 100 a cycle; 12 cycles a column for the results of the last one, and of pairs to take the sums out; parts of K
// 2500 and 8 a column, where their clusters fit the machine at once (five steps of 200 x 2000 float32 took 188 us in parts and 248 without, of 1031 x 602
// 206 and 236, of 500 x 500 181 and 197, of 200 x 2000 bfloat16 148 and 166, before the code that stores results was made shorter).
static Tiling tiling(const int planes_a, const int planes_b, int64_t m, int64_t n, int64_t k, int64_t batch, bool symmetric, bool wide, int64_t p, int sms) {
  const int products = planes_a + planes_b - 1, chunks = chunks_of(wide, p);
  Tiling best{1, 64, 1};
  int64_t least = 0;
  for (const Tiling t : {Tiling{2, 256, 1}, Tiling{2, 128, 1}, Tiling{1, 256, 1}, Tiling{1, 128, 1}, Tiling{1, 64, 1}, Tiling{1, 128, 4}, Tiling{1, 128, 2}, Tiling{1, 64, 2}}) {
    if (wide && t.columns > kMaxSums) continue;
    const int64_t total = tiles(m, n, kM * t.ctas, t.columns, symmetric && t.split == 1) * batch, rounds = ceil_div(total, sms / t.ctas);
    const int64_t all = ceil_div(k, kK * chunks), steps = ceil_div(all, t.split);
    if (t.split > 1 && (total * t.split > sms * 7 / 8 || all < 2 * t.split)) continue;
    const int64_t mma = products * chunks * 4 * (t.columns / 2 > 46 ? t.columns / 2 : 46), bytes = (int64_t)chunks * 128 * (kM * planes_a + t.columns / t.ctas * planes_b);
    int64_t step = mma > bytes / 100 ? mma : bytes / 100;
    const int64_t issue = products * chunks * 4 * 46 + (wide ? 400 : 250), taken = wide ? 250 + 3 * t.columns : 0;
    if (step < issue) step = issue;
    if (step < taken) step = taken;
    const int64_t cycles = rounds * (steps * step + (wide ? 12 * t.columns : 0)) + 12 * t.columns / t.split + (t.split > 1 ? 2500 + 8 * t.columns : 0);
    if (least != 0 && cycles >= least) continue;
    least = cycles;
    best = t;
  }
  return best;
}

struct Product {
  Planes a, b;
  int a_planes, b_planes, a_turned, b_turned;
  int64_t a_rows, a_cols, a_ld, b_rows, b_cols, b_ld;  // the operands' matrices as they lie
  int64_t m, n, k;
  bool symmetric;
  int64_t smaller = 0;                 // side of the matrices
};

template <int MODE, typename T>
static int multiply(const char* op, const Product& x, Params p, const Matrices& s, int64_t batch, cudaStream_t st) {
  const int sms = current_sm_count();
  p.m = (int)x.m; p.n = (int)x.n;
  p.chunks = chunks_of(is_wide<T>, x.smaller);
  p.steps = (int)ceil_div(x.k, kK * p.chunks);
  p.batch = (int)batch;
  const Tiling shape = tiling(x.a_planes, x.b_planes, x.m, x.n, x.k, batch, x.symmetric, is_wide<T>, x.smaller, sms);
  p.split = shape.split;
  p.a = Operand{kM, x.a_turned, x.a_planes};
  p.b = Operand{shape.columns / shape.ctas, x.b_turned, x.b_planes};
  p.col_tiles = (int)ceil_div(x.n, shape.columns);
  // (where all tiles are done at once, the half of them would save nothing but cost the second writing)
  p.symmetric = x.symmetric && tiles(x.m, x.n, kM * shape.ctas, shape.columns, false) * batch > sms / shape.ctas;
  p.items = (int)tiles(x.m, x.n, kM * shape.ctas, shape.columns, p.symmetric != 0);
  const int64_t total = (int64_t)p.items * batch, places = sms / (shape.ctas * shape.split);
  F2C_REQUIRE(total < (1ll << 30), F2C_ERR_LIMIT, "%s: too many tiles", op);
  const unsigned grid = (unsigned)((total < places ? total : places) * shape.ctas * shape.split);
  p.issued = p.issued ? (int)total : 0;
  p.error = stream_error_word();
  const size_t stage = (size_t)p.a.bytes(p.chunks) * p.a.planes + (size_t)p.b.bytes(p.chunks) * p.b.planes, parts = shape.split > 1 ? (size_t)shape.columns * kM * 4 : 0;
  p.stages = (int)((kRoom - 1024 - parts) / stage);
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.parts_at = (int)(p.stages * stage);
  Maps maps;
  const __half* ap[2] = {x.a.high, x.a.low};
  const __half* bp[2] = {x.b.high, x.b.low};
  bool ok = true;
  for (int q = 0; q < 2; ++q) {
    ok = ok && make_stack_map(maps.a + q, ap[q < x.a_planes ? q : 0], batch, x.a_rows, x.a_cols, 2 * x.a_ld, x.a_turned ? kK * p.chunks : kM);
    ok = ok && make_stack_map(maps.b + q, bp[q < x.b_planes ? q : 0], batch, x.b_rows, x.b_cols, 2 * x.b_ld, x.b_turned ? kK * p.chunks : p.b.rows);
  }
  F2C_REQUIRE(ok, F2C_ERR_CUDA, "%s: tensor map", op);
  auto* kern = shape.ctas == 2 ? product_kernel<MODE, T, 2, false> : shape.split > 1 ? product_kernel<MODE, T, 1, true> : product_kernel<MODE, T, 1, false>;
  if (const int rc = allow_smem(op, (const void*)kern, (int)kRoom)) return rc;
  launch_dependent_cluster(kern, dim3(grid), kThreads, p.stages * stage + parts + 1024, (unsigned)(shape.ctas * shape.split), st, maps, p, s);
  return check_launch(op);
}

template <typename T>
static int run_typed(const char* op, Matrices& src, const Shape& s, const Steps& st, char* ws, cudaStream_t stream) {
  constexpr bool kWide = is_wide<T>;
  const bool exact = sizeof(T) == 2 && src.listed == 0, tall = s.rows > s.cols;
  auto take = [&](int64_t bytes) { char* at = ws; ws += bytes; return at; };
  Planes x[2], a{}, r{};
  for (Planes& q : x) { q.high = (__half*)take(s.x_bytes()); q.low = (__half*)take(s.x_bytes()); }
  for (Planes* q : {&a, &r}) { q->high = (__half*)take(s.p_bytes()); q->low = s.fine(kWide) ? (__half*)take(s.p_bytes()) : nullptr; }
  double* parts = (double*)take(round256(8 * s.batch * kMaxParts));
  Factors* table = (Factors*)take(0);
  src.size = s.rows * s.cols;
  bool four = s.cols % 4 == 0 && aligned(src.g, 4 * sizeof(T));
  for (int i = 0; i < src.listed; ++i) four = four && aligned(src.list[i].grad, 4 * sizeof(T)) && aligned(src.list[i].momentum, 16);
  // 16 elements a thread, more of matrices over 4 M elements
  int64_t cut = ceil_div(src.size, 16 * kLoadThreads);
  if (cut > kMaxParts) cut = kMaxParts;
  const dim3 grid((unsigned)cut, (unsigned)s.batch);
  int planes = st.count == 0 ? (exact ? 1 : 2) : x_planes(st, 0, kWide, exact);
  __half* low = planes > 1 ? x[0].low : nullptr;
  if (four) {
    launch_dependent(norm_kernel<T, 4>, grid, kLoadThreads, 0, stream, src, parts);
    launch_dependent(planes_kernel<T, 4>, grid, kLoadThreads, 0, stream, src, st, (const double*)parts, x[0].high, low, s.rows, s.cols, s.ldx(), table);
  } else {
    launch_dependent(norm_kernel<T, 1>, grid, kLoadThreads, 0, stream, src, parts);
    launch_dependent(planes_kernel<T, 1>, grid, kLoadThreads, 0, stream, src, st, (const double*)parts, x[0].high, low, s.rows, s.cols, s.ldx(), table);
  }
  if (const int rc = check_launch(op)) return rc;
  if (st.count == 0) {
    launch_dependent(store_kernel<T>, grid, kLoadThreads, 0, stream, src, (const __half*)x[0].high, (const __half*)low, s.rows, s.cols, s.ldx(), (const Factors*)table);
    return check_launch(op);
  }
  const int64_t p = s.p();
  const int gram_planes = kWide ? 2 : 1, inner = s.fine(kWide) ? 2 : 1;  // of X in A = X X^T, and of A and R
  for (int t = 0; t < st.count; ++t) {
    const bool last = t + 1 == st.count, poly = st.co[3 * t + 2] != 0.0f;
    // A = X X^T: of a tall matrix, whose transpose X is, the rows run along K
    Product gram{x[t & 1], x[t & 1], gram_planes, gram_planes, tall, tall, s.rows, s.cols, s.ldx(), s.rows, s.cols, s.ldx(), p, p, tall ? s.rows : s.cols, true};
    Params g{};
    g.factors = table + t;
    g.issued = st.tries != 0u;
    g.high = poly ? a.high : r.high; g.low = poly ? a.low : r.low;
    g.ld = s.ldp(); g.stack = p * s.ldp();
    gram.smaller = p;
    if (const int rc = multiply<kGram, T>(op, gram, g, src, s.batch, stream)) return rc;
    if (poly) {
      Product square{a, a, inner, inner, 0, 0, p, p, s.ldp(), p, p, s.ldp(), p, p, p, true};
      Params q = g;
      q.add_high = a.high; q.add_low = a.low;
      q.high = r.high; q.low = r.low;
      square.smaller = p;
      if (const int rc = multiply<kPoly, T>(op, square, q, src, s.batch, stream)) return rc;
    }
    // the rows of the next X are columns of this product, so that a warp writes 32 neighbours
    const int next = last ? 1 : x_planes(st, t + 1, kWide, exact);
    Product apply = tall ? Product{r, x[t & 1], inner, planes, 0, 0, p, p, s.ldp(), s.rows, s.cols, s.ldx(), p, s.rows, p, false}
                         : Product{x[t & 1], r, planes, inner, 1, 0, s.rows, s.cols, s.ldx(), p, p, s.ldp(), s.cols, p, p, false};
    apply.smaller = p;
    Params q{};
    q.factors = table + t;
    q.issued = st.tries != 0u;
    q.gain = src.lr * (float)sqrt(s.rows > s.cols ? (double)s.rows / (double)s.cols : 1.0);
    q.add_high = x[t & 1].high; q.add_low = planes > 1 ? x[t & 1].low : nullptr;
    q.high = x[(t + 1) & 1].high; q.low = next > 1 ? x[(t + 1) & 1].low : nullptr;
    q.ld = s.ldx(); q.stack = s.rows * s.ldx();
    if (const int rc = last ? multiply<kFinal, T>(op, apply, q, src, s.batch, stream) : multiply<kApply, T>(op, apply, q, src, s.batch, stream)) return rc;
    planes = next;
  }
  return F2C_OK;
}

static int run(const char* op, Matrices& src, int dtype, const Shape& s, const Steps& st, char* ws, cudaStream_t stream) {
  if (is_small(s.rows, s.cols)) {
    src.size = s.rows * s.cols;
    return small(op, src, (int)s.batch, s.rows, s.cols, dtype, st, stream);
  }
  if (dtype == F2C_F32) return run_typed<float>(op, src, s, st, ws, stream);
  if (dtype == F2C_F16) return run_typed<__half>(op, src, s, st, ws, stream);
  return run_typed<__nv_bfloat16>(op, src, s, st, ws, stream);
}

// Singular values start in [0, 1].  What keeps the half-precision operands in range: no step may take one out of [0, 7.9], and R has none over 60.
static int check(const char* op, int dtype, const float* co, int steps, float eps, Steps* st) {
  F2C_REQUIRE(is_float_dtype(dtype), F2C_ERR_UNSUPPORTED, "%s: matrices must be float32, float16 or bfloat16", op);
  st->tries = steps & F2C_NO_WAITS ? 0u : kWaitLimit;
  steps &= ~F2C_NO_WAITS;
  F2C_REQUIRE(steps >= 0 && steps <= F2C_MAX_NS_STEPS, F2C_ERR_LIMIT, "%s: 0 to %d steps", op, F2C_MAX_NS_STEPS);
  F2C_REQUIRE(steps == 0 || co, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(eps >= 0.0f && eps <= 3.4028235e38f, F2C_ERR_INVALID, "%s: eps must not be negative", op);
  st->count = steps;
  st->eps = eps;
  double top = 1.0;
  st->top[0] = 1.0f;
  for (int t = 0; t < steps; ++t, co += 3) {
    double factor = 0.0, next = 0.0, r = 0.0;
    for (int i = 0; i <= 1024; ++i) {
      const double v = top * i / 1024, w = v * v * (co[1] + v * v * co[2]), f = fabs(co[0] + w);
      if (!(fabs(w) <= r)) r = fabs(w);
      if (!(f <= factor)) factor = f;
      if (!(v * f <= next)) next = v * f;
    }
    F2C_REQUIRE(r <= 60.0 && next <= 7.9, F2C_ERR_LIMIT, "%s: the coefficients of step %d let the matrix grow too far", op, t);
    top = next;
    for (int i = 0; i < 3; ++i) st->co[3 * t + i] = co[i];
    st->factor[t] = (float)factor;
    st->top[t + 1] = (float)top;
  }
  return F2C_OK;
}

static int check_shape(const char* op, const Shape& s) {
  F2C_REQUIRE(s.batch >= 0 && s.rows >= 0 && s.cols >= 0, F2C_ERR_INVALID, "%s: negative size", op);
  F2C_REQUIRE(s.batch <= 65535 && s.rows <= 65536 && s.cols <= 65536, F2C_ERR_LIMIT, "%s: at most 65535 matrices of 65536 rows and columns", op);
  return F2C_OK;
}

}  // namespace ns
}  // namespace f2c

using namespace f2c;

extern "C" int64_t f2c_orthogonalize_workspace(int dtype, int64_t batch, int64_t rows, int64_t cols) {
  return batch < 1 || rows < 1 || cols < 1 || ns::is_small(rows, cols) ? 0 : ns::workspace(ns::Shape{batch, rows, cols}, dtype != F2C_BF16);
}

extern "C" int f2c_orthogonalize(const void* g, void* out, int dtype, int64_t batch, int64_t rows, int64_t cols, const float* coefficients_host,
                                 int steps, float eps, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "orthogonalize";
  const ns::Shape s{batch, rows, cols};
  ns::Steps st{};
  if (const int rc = ns::check_shape(op, s)) return rc;
  if (const int rc = ns::check(op, dtype, coefficients_host, steps, eps, &st)) return rc;
  if (batch == 0 || rows == 0 || cols == 0) return F2C_OK;
  F2C_REQUIRE(g && out, F2C_ERR_INVALID, "%s: null pointer", op);
  const uintptr_t from = (uintptr_t)g, to = (uintptr_t)out, bytes = (uintptr_t)batch * (uintptr_t)rows * (uintptr_t)cols * dtype_size(dtype);
  F2C_REQUIRE(from == to || from + bytes <= to || to + bytes <= from, F2C_ERR_INVALID, "%s: out shares a part of g's memory", op);
  const int64_t need = f2c_orthogonalize_workspace(dtype, batch, rows, cols);
  F2C_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), F2C_ERR_INVALID,
              "%s: workspace too small or not 256-byte aligned", op);
  ns::Matrices src{};
  src.g = g;
  src.out = out;
  return ns::run(op, src, dtype, s, st, (char*)workspace, (cudaStream_t)stream);
}

// The matrices that are done together with number i of the list, from it on, up to kMaxList: all small ones, or those of its shape.  False when an earlier
// one was their first.
static bool group_of(const f2c_muon_matrix* list, int count, int i, ns::Matrices* src) {
  const bool small = ns::is_small(list[i].rows, list[i].cols);
  const auto with = [&](int j) {
    if (list[j].rows == 0 || list[j].cols == 0) return false;
    return small ? ns::is_small(list[j].rows, list[j].cols) : list[j].rows == list[i].rows && list[j].cols == list[i].cols;
  };
  if (list[i].rows == 0 || list[i].cols == 0) return false;
  int before = 0;
  for (int j = 0; j < i; ++j) before += with(j);
  if (before % ns::kMaxList != 0) return false;
  src->listed = 0;
  for (int j = i; j < count && src->listed < ns::kMaxList; ++j)
    if (with(j)) src->list[src->listed++] = list[j];
  return true;
}

// Whether anything of the list that is written shares memory with anything else of it: the matrices of a launch are worked on at the same time.
static bool overlaps(const f2c_muon_matrix* list, int count, int dtype) {
  struct Range { uintptr_t from, to; bool written; };
  std::vector<Range> all;
  all.reserve(3 * (size_t)count);
  for (int i = 0; i < count; ++i) {
    const f2c_muon_matrix& m = list[i];
    const uintptr_t size = (uintptr_t)m.rows * (uintptr_t)m.cols;
    if (size == 0) continue;
    const auto put = [&](const void* p, size_t item, bool written) { all.push_back(Range{(uintptr_t)p, (uintptr_t)p + size * item, written}); };
    put(m.weight, dtype_size(dtype), true);
    put(m.grad, dtype_size(dtype), false);
    put(m.momentum, 4, true);
  }
  std::sort(all.begin(), all.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
  uintptr_t end = 0, written_end = 0;  // of those that begin before
  for (const Range& r : all) {
    if (r.from < (r.written ? end : written_end)) return true;
    end = std::max(end, r.to);
    if (r.written) written_end = std::max(written_end, r.to);
  }
  return false;
}

extern "C" int64_t f2c_muon_workspace(const f2c_muon_matrix* list_host, int count, int dtype) {
  int64_t most = 0;
  ns::Matrices src{};
  for (int i = 0; list_host != nullptr && i < count; ++i) {
    if (list_host[i].rows < 0 || list_host[i].cols < 0 || ns::is_small(list_host[i].rows, list_host[i].cols) || !group_of(list_host, count, i, &src)) continue;
    const int64_t bytes = ns::workspace(ns::Shape{src.listed, list_host[i].rows, list_host[i].cols}, dtype != F2C_BF16);
    most = bytes > most ? bytes : most;
  }
  return most;
}

extern "C" int f2c_muon_step(const f2c_muon_matrix* list_host, int count, int dtype, float lr, float momentum, int nesterov, float decay,
                             const float* coefficients_host, int steps, float eps, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "muon_step";
  ns::Steps st{};
  F2C_REQUIRE(count >= 0 && (count == 0 || list_host), F2C_ERR_INVALID, "%s: bad list", op);
  if (const int rc = ns::check(op, dtype, coefficients_host, steps, eps, &st)) return rc;
  for (int i = 0; i < count; ++i) {
    const f2c_muon_matrix& m = list_host[i];
    if (const int rc = ns::check_shape(op, ns::Shape{1, m.rows, m.cols})) return rc;
    F2C_REQUIRE(m.rows == 0 || m.cols == 0 || (m.weight && m.grad && m.momentum), F2C_ERR_INVALID, "%s: null pointer", op);
  }
  try {
    F2C_REQUIRE(!overlaps(list_host, count, dtype), F2C_ERR_INVALID, "%s: a weight or momentum shares memory with another tensor of the step", op);
  } catch (...) {
    return set_error(F2C_ERR_LIMIT, "%s: no host memory for a list of %d matrices", op, count);
  }
  const int64_t need = f2c_muon_workspace(list_host, count, dtype);
  F2C_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), F2C_ERR_INVALID,
              "%s: workspace too small or not 256-byte aligned", op);
  ns::Matrices src{};
  src.mu = momentum;
  src.keep = (float)(1.0 - (double)lr * decay);
  src.lr = lr;
  src.nesterov = nesterov;
  for (int i = 0; i < count; ++i) {
    if (!group_of(list_host, count, i, &src)) continue;
    const ns::Shape s{src.listed, list_host[i].rows, list_host[i].cols};
    if (const int rc = ns::run(op, src, dtype, s, st, (char*)workspace, (cudaStream_t)stream)) return rc;
  }
  return F2C_OK;
}
