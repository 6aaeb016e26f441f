// Gradient of a linear layer's weight and bias, its input kept in 8 bits (f2c_checkpoint_weight_grad):
//   dW[i, j] = sum over rows r of dy[r, i] (low[r, g] + step[r, g] q[r, j]),   db[i] = sum over rows of dy[r, i],   g the group of column j,
// on the 5th-generation tensor cores.  The input is never written out: with the factors taken to the other side,
//   dW = (step dy)^T q + (low dy)^T 1,
// the codes q = 0 .. 255 are bfloat16 numbers as they are, and step dy, rounded to single precision, is a sum of bfloat16 numbers: three of them hold
// all 24 bits (float32 dy), two 16 (float16 and bfloat16 dy, whose result is rounded to 11 or 8).  The second term is one number for every i and
// group, summed in registers on the way, as is db.
//
// A tile of dW has 128 columns of dy (the lanes of TMEM) and a group's 128 columns of q, so that all of a row's tile has one step.  Neither operand is
// turned: their rows run along M and N, which the MMA takes as it is.  Sixteen warps load 32 rows of both, two stages ahead in registers, and
// write them as bfloat16 to a ring in shared memory; the first of them also issues the MMAs, of a stage when it has written its part of the next (a
// warp of its own would leave the others 96 registers instead of 128).
//
// Sums.  The tensor cores cut sums off instead of rounding them, for every 16 rows.  So for float32 the two small parts of step dy have an
// accumulator of their own, and sums are taken out every 256 rows and added up in registers, while the MMAs go on in the other half of TMEM.
//
// Many rows and few tiles: the rows are dealt out over all SMs; each leaves its part of the sums, and a second launch adds them up in their order.
#include <algorithm>
#include <type_traits>

#include "checkpoint.cuh"
#include "tcgen05.cuh"

namespace f2c {
namespace wg {

using namespace t5;
using ckpt::fma2;
using ckpt::kGroup;
using ckpt::mul2;
using ckpt::pair_of;

constexpr int kWarps = 16, kThreads = 32 * kWarps;
constexpr int kTile = 128, kRows = 32, kAhead = 2, kStages = 6;
constexpr uint32_t kChunk = kRows * 128, kPlane = 2 * kChunk;  // 64 columns' rows, and a tile's
constexpr uint32_t kFormatBf16 = 1;

struct Params {
  const void* dy;
  int64_t ldy, m;
  int n, k;
  ckpt::Codes x;
  int n_tiles, splits;
  int64_t split_rows;     // a multiple of kRows
  void *dw, *db;          // (splits == 1) of dy's type
  float *part, *part_db;  // (splits > 1) [split][tile][32][128][4], [split][n_tiles * 128]
  uint32_t tries;
  int* error;
};

struct Bars {
  uint64_t full[kStages], empty[kStages], drain, acc_full[2], acc_empty[2];
  uint32_t tmem;
  int failed;
};

template <typename T> struct Kind { static constexpr int kPieces = 2, kTaken = 128; };  // stages between two takings out
template <> struct Kind<float> { static constexpr int kPieces = 3, kTaken = 8; };
static_assert(Kind<float>::kTaken >= kStages, "a ring's stages do not reach over two takings out");

__device__ __forceinline__ uint32_t pack_bf16(float low, float high) {  // round to even
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(high), "f"(low));
  return r;
}
__device__ __forceinline__ void store16(uint32_t at, const uint32_t (&w)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}

// What a thread has of a stage: eight columns of a row of dy and of its codes, and their step and lowest value.  ACCESS: bytes of a load of dy.
template <typename T, int ACCESS>
struct Piece {
  static constexpr int kWords = 2 * (int)sizeof(T), kEach = ACCESS / (int)sizeof(T);
  uint32_t dy[kWords];
  uint2 codes, scale;

  __device__ __forceinline__ void load(const Params& p, int64_t row, bool here, int col, int code_col, int group) {
    const T* const from = (const T*)p.dy + row * p.ldy + col;
#pragma unroll
    for (int q = 0; q < 8 / kEach; ++q) {
      const bool go = here && col + q * kEach < p.n;
      const T* const at = from + q * kEach;
      if constexpr (ACCESS == 16) {
        const uint4 v = ldg_nc_u128_if(at, go);
        dy[4 * q] = v.x; dy[4 * q + 1] = v.y; dy[4 * q + 2] = v.z; dy[4 * q + 3] = v.w;
      } else if constexpr (ACCESS == 8) {
        const uint2 v = ldg_nc_u64_if(at, go);
        dy[2 * q] = v.x; dy[2 * q + 1] = v.y;
      } else if constexpr (ACCESS == 4) {
        dy[q] = ldg_nc_u32_if(at, go);
      } else {
        const uint32_t v = go ? (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(at)) : 0u;
        dy[q / 2] = q & 1 ? dy[q / 2] | v << 16 : v;
      }
    }
    codes = ldg_nc_u64_if(p.x.codes + row * p.x.ld + code_col, here && code_col < p.k);
    scale = ldg_nc_u64_if(p.x.scales + 2 * (row * p.x.groups + group), here);
  }
  __device__ __forceinline__ void get(unsigned long long (&d)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (sizeof(T) == 4) d[e] = pair_of(__uint_as_float(dy[2 * e]), __uint_as_float(dy[2 * e + 1]));
      else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&dy[e]));
        d[e] = pair_of(f.x, f.y);
      } else {
        d[e] = pair_of(__uint_as_float(dy[e] << 16), __uint_as_float(dy[e] & 0xffff0000u));
      }
    }
  }
};

template <typename T, int ACCESS>
__global__ void __launch_bounds__(kThreads, 1) weight_grad_kernel(const __grid_constant__ Params p) {
  constexpr int kPieces = Kind<T>::kPieces, kTaken = Kind<T>::kTaken;
  constexpr uint32_t kStage = (kPieces + 1) * kPlane;
  constexpr uint32_t kAcc = kPieces == 3 ? 256 : 128;  // columns of TMEM: the sums, and those of the small parts
  extern __shared__ unsigned char smem_raw[];
  __shared__ Bars bars;
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  const int tile = (int)blockIdx.x / p.splits, split = (int)blockIdx.x % p.splits, n0 = tile % p.n_tiles * kTile, group = tile / p.n_tiles;
  const int64_t row0 = split * p.split_rows, rows = min(p.split_rows, p.m - row0);
  const int stages = (int)((rows + kRows - 1) / kRows), takes = (stages + kTaken - 1) / kTaken;
  uint32_t left = p.tries;

  if (wid == 0) alloc_tmem(&bars.tmem, 2 * kAcc);
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) { init_bar(bars.full + s, kWarps); init_bar(bars.empty + s, 1); }
    init_bar(&bars.drain, 1);
    for (int b = 0; b < 2; ++b) { init_bar(bars.acc_full + b, 1); init_bar(bars.acc_empty + b, kWarps); }
    fence_bars();
    bars.failed = 0;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = bars.tmem;
  dependency_wait();
  release_dependents();

  float sum[32];
  unsigned long long of_low[4], of_bias[4];  // the tile's sums that this thread has, and over its rows and eight columns
#pragma unroll
  for (int j = 0; j < 32; ++j) sum[j] = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) of_low[e] = of_bias[e] = 0ull;
  const int vec = tid & 15, at_row = tid >> 4;  // eight columns, and a row of a stage
  const int col = n0 + 8 * vec, code_col = group * kGroup + 8 * vec;
  // 16 bytes `vec` of row at_row, in the 128-byte swizzle
  const uint32_t place = smem_u32(smem) + (uint32_t)(vec >> 3) * kChunk + (uint32_t)at_row * 128 + (uint32_t)(((vec & 7) ^ (at_row & 7)) << 4);
  const int quarter = wid & 3, cols = wid >> 2;
  const uint32_t acc_at = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)cols * 32;

  // ================= sums of kTaken stages out of TMEM
  const auto take = [&](int t) {
    wait_bar(bars.acc_full + (t & 1), (t >> 1) & 1, left);
    fence_after();
#pragma unroll
    for (int part = 0; part < (kPieces == 3 ? 2 : 1); ++part) {
      uint32_t r[32];
      tmem_ld32(acc_at + (uint32_t)(t & 1) * kAcc + part * 128, r);
      tmem_wait(r);
#pragma unroll
      for (int j = 0; j < 32; ++j) sum[j] += __uint_as_float(r[j]);
    }
    fence_before();
    __syncwarp();
    if (lane == 0) arrive(bars.acc_empty + (t & 1));
  };

  // ================= MMAs of stage i, whose place in the ring is s
  const bool mine = wid == 0 && elected() != 0u;
  const uint32_t idesc = instruction(kSumF32, kFormatBf16, kTile, kTile) | kTurnedA | kTurnedB;
  const uint32_t a_low = desc_low(smem_u32(smem), kChunk), b_low = a_low + (kPieces * kPlane >> 4);
  const auto multiply = [&](int i, int s, uint32_t round) {
    const int t = i / kTaken, in_take = i % kTaken;
    const uint32_t acc = tmem + (uint32_t)(t & 1) * kAcc;
    if (in_take == 0 && t >= 2) wait_bar(bars.acc_empty + (t & 1), ((t >> 1) - 1) & 1, left);
    wait_bar(bars.full + s, round & 1, left);
    fence_after();
    const bool go = mine && left != 0u;
    const uint32_t at = (uint32_t)s * (kStage >> 4), a = a_low + at, b = b_low + at;
#pragma unroll
    for (uint32_t q = 0; q < kRows / 16; ++q) {
      mma_f16(go, acc, desc(a + q * kStepTurned), desc(b + q * kStepTurned), idesc, in_take != 0 || q != 0);
#pragma unroll
      for (uint32_t piece = 1; piece < kPieces; ++piece)
        mma_f16(go, kPieces == 3 ? acc + 128 : acc, desc(a + piece * (kPlane >> 4) + q * kStepTurned), desc(b + q * kStepTurned), idesc,
                kPieces == 2 || in_take != 0 || q != 0 || piece != 1);
    }
    commit(go, bars.empty + s);
    if (in_take == kTaken - 1 || i == stages - 1) commit(go, bars.acc_full + (t & 1));
    __syncwarp();
  };

  // ================= dy and codes, as the MMAs take them
  const auto fetch = [&](Piece<T, ACCESS>& v, int i) {
    const int64_t r = (int64_t)i * kRows + at_row;
    v.load(p, row0 + r, r < rows, col, code_col, group);
  };
  Piece<T, ACCESS> ahead[kAhead];
#pragma unroll
  for (int a = 0; a < kAhead; ++a) fetch(ahead[a], a);
  int s = 0, taken = 0;
  uint32_t round = 0;
  for (int i0 = 0; i0 < stages; i0 += kAhead) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int i = i0 + a;
      if (i >= stages) break;
      const Piece<T, ACCESS> v = ahead[a];
      fetch(ahead[a], i + kAhead);
      unsigned long long d[4];
      v.get(d);
      if (group == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) add2(of_bias[e], d[e]);
      }
      const unsigned long long step = pair_of(__uint_as_float(v.scale.x), __uint_as_float(v.scale.x)), low = pair_of(__uint_as_float(v.scale.y), __uint_as_float(v.scale.y));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        of_low[e] = fma2(low, d[e], of_low[e]);
        d[e] = mul2(step, d[e]);
      }
      if (round > 0) wait_bar(bars.empty + s, (round - 1) & 1, left);
      const uint32_t at = place + (uint32_t)s * kStage;
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = pack_bf16(lo32(d[e]), hi32(d[e]));
          // what is left: exact
          if (q + 1 < kPieces) d[e] = fma2(pair_of(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u)), pair_of(-1.0f, -1.0f), d[e]);
        }
        store16(at + (uint32_t)q * kPlane, w);
      }
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // 2^23 + q, less 2^23
        const uint32_t from = e < 2 ? v.codes.x : v.codes.y;
        unsigned long long q = pair_of(__uint_as_float(__byte_perm(from, 0x4B000000u, 0x7440 + (e & 1) * 2)), __uint_as_float(__byte_perm(from, 0x4B000000u, 0x7441 + (e & 1) * 2)));
        add2(q, pair_of(-8388608.0f, -8388608.0f));
        w[e] = pack_bf16(lo32(q), hi32(q));
      }
      store16(at + kPieces * kPlane, w);
      fence_async();
      __syncwarp();
      if (lane == 0) arrive(bars.full + s);
      if (wid == 0 && i > 0) multiply(i - 1, s > 0 ? s - 1 : kStages - 1, s > 0 ? round : round - 1);
      if (++s == kStages) { s = 0; ++round; }
      // the sums are ready some time after the last of their stages has been handed over
      if ((taken + 1) * kTaken + kStages <= i + 1) take(taken++);
    }
  }
  if (wid == 0 && stages > 0) multiply(stages - 1, s > 0 ? s - 1 : kStages - 1, s > 0 ? round : round - 1);
  while (taken < takes) take(taken++);
  if (left == 0u) bars.failed = 1;
  fence_before();
  __syncthreads();
  const bool lost = bars.failed != 0;
  if (lost && p.tries != 0u) {
    // MMAs in flight read shared memory and write TMEM: wait (bounded) for what was issued
    left = p.tries;
    if (wid == 0) {
      commit(mine, &bars.drain);
      wait_bar(&bars.drain, 0, left);
    }
    __syncthreads();
  }
  if (wid == 0) {
    fence_after();
    free_tmem(tmem, 2 * kAcc);
  }
  if (tid == 0 && lost) report_wait(p.error, 8);

  // of_low and of_bias over all rows: the ring's memory is free
  float(*const columns)[2][kTile] = reinterpret_cast<float(*)[2][kTile]>(smem);  // [warp]
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    add2(of_low[e], __shfl_xor_sync(0xffffffffu, of_low[e], 16));
    add2(of_bias[e], __shfl_xor_sync(0xffffffffu, of_bias[e], 16));
  }
  if (lane < 16) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      *reinterpret_cast<unsigned long long*>(&columns[wid][0][8 * lane + 2 * e]) = of_low[e];
      *reinterpret_cast<unsigned long long*>(&columns[wid][1][8 * lane + 2 * e]) = of_bias[e];
    }
  }
  __syncthreads();
  if (tid < 2 * kTile) {
    float all = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) all += columns[w][tid >> 7][tid & 127];
    columns[0][tid >> 7][tid & 127] = all;  // (read by this thread alone)
  }
  __syncthreads();
  const int i = quarter * 32 + lane;
  const float more = lost ? __int_as_float(0x7fffffff) : columns[0][0][i];
#pragma unroll
  for (int j = 0; j < 32; ++j) sum[j] += more;
  if (p.splits > 1) {
    float4* const to = reinterpret_cast<float4*>(p.part) + ((int64_t)split * (gridDim.x / p.splits) + tile) * (kTile * kTile / 4) + cols * 8 * kTile + i;
#pragma unroll
    for (int j = 0; j < 8; ++j) to[j * kTile] = make_float4(sum[4 * j], sum[4 * j + 1], sum[4 * j + 2], sum[4 * j + 3]);
    if (group == 0 && tid < kTile) p.part_db[(int64_t)split * p.n_tiles * kTile + n0 + tid] = columns[0][1][tid];
    return;
  }
  if (n0 + i < p.n) {
    const int first = group * kGroup + cols * 32, count = p.k - first;
    T* const to = (T*)p.dw + (int64_t)(n0 + i) * p.k + first;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < count) to[j] = from_float<T>(sum[j]);
  }
  if (group == 0 && tid < kTile && n0 + tid < p.n) ((T*)p.db)[n0 + tid] = from_float<T>(columns[0][1][tid]);
}

// Adds the parts up: 32 columns of dy and four of q to a CTA, an eighth of the parts to a warp.  Behind the tiles' CTAs those of db.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Params p, int tiles) {
  __shared__ float4 of[8][33];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per_tile = kTile * kTile / 128;
  const bool bias = (int)blockIdx.x >= tiles * per_tile;
  if (bias) {
    const int i = ((int)blockIdx.x - tiles * per_tile) * 32 + lane;
    float sum = 0.0f;
    for (int s = warp; s < p.splits; s += 8) sum += p.part_db[(int64_t)s * p.n_tiles * kTile + i];
    of[warp][lane].x = sum;
    __syncthreads();
    if (warp != 0 || i >= p.n) return;
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += of[w][lane].x;
    ((T*)p.db)[i] = from_float<T>(sum);
    return;
  }
  const int tile = blockIdx.x / per_tile, rest = blockIdx.x % per_tile, quad = rest / 4, i = rest % 4 * 32 + lane;
  const float4* const from = reinterpret_cast<const float4*>(p.part) + (int64_t)tile * (kTile * kTile / 4) + quad * kTile + i;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int s = warp; s < p.splits; s += 8) {
    const float4 v = from[(int64_t)s * tiles * (kTile * kTile / 4)];
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  }
  of[warp][lane] = sum;
  __syncthreads();
  const int n = tile % p.n_tiles * kTile + i, col = tile / p.n_tiles * kGroup + quad * 4;
  if (warp != 0 || n >= p.n) return;
  sum = of[0][lane];
#pragma unroll
  for (int w = 1; w < 8; ++w) {
    const float4 v = of[w][lane];
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  }
  T* const to = (T*)p.dw + (int64_t)n * p.k + col;
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < p.k) to[e] = from_float<T>(v[e]);
}

struct Plan {
  int n_tiles, k_tiles, splits;
  int64_t split_rows, part_bytes, bytes;
};

// How many ways the rows are split: the choice of least time, in cycles: a stage takes an SM 600, a tile's start and end 5000, the parts' way through
// L2 and back 64 KB each at 4000 bytes a cycle for all SMs, and the launch that adds them up 4000.
static Plan plan(int64_t m, int64_t n, int64_t k) {
  Plan p{};
  p.n_tiles = (int)ceil_div(n, kTile);
  p.k_tiles = (int)ceil_div(k, kGroup);
  const int64_t tiles = (int64_t)p.n_tiles * p.k_tiles, stages = ceil_div(m, kRows);
  int64_t least = INT64_MAX;
  for (int64_t s = 1; s <= std::min<int64_t>(stages, kSmCount); ++s) {
    if (s > 1 && tiles * s > 2 * kSmCount) break;
    const int64_t each = ceil_div(stages, s);
    if (s > 1 && ceil_div(stages, each) != s) continue;  // (the last ones would have none)
    const int64_t cycles = ceil_div(tiles * s, kSmCount) * (each * 600 + 5000) + (s > 1 ? 4000 + tiles * s * 2 * 65536 / 4000 : 0);
    if (cycles >= least) continue;
    least = cycles;
    p.splits = (int)s;
    p.split_rows = each * kRows;
  }
  if (p.splits > 1) {
    p.part_bytes = tiles * p.splits * kTile * kTile * 4;
    p.bytes = p.part_bytes + ceil_div((int64_t)p.splits * p.n_tiles * kTile * 4, 256) * 256;
  }
  return p;
}

template <typename T, int ACCESS>
static int run(const char* op, const Params& p, const Plan& how, cudaStream_t st) {
  constexpr int bytes = kStages * (Kind<T>::kPieces + 1) * kPlane + 1024;
  const int tiles = how.n_tiles * how.k_tiles;
  if (const int rc = allow_smem(op, (const void*)weight_grad_kernel<T, ACCESS>, bytes)) return rc;
  launch_dependent(weight_grad_kernel<T, ACCESS>, dim3((unsigned)(tiles * how.splits)), kThreads, bytes, st, p);
  if (how.splits > 1) launch_dependent(join_kernel<T>, dim3((unsigned)(tiles * (kTile * kTile / 128) + how.n_tiles * 4)), 256, 0, st, p, tiles);
  return check_launch(op);
}

// by the widest loads that dy's rows allow
template <typename T>
static int run(const char* op, const Params& p, const Plan& how, cudaStream_t st) {
  int access = 16;
  const int64_t item = sizeof(T);
  while (access > item && (!aligned(p.dy, access) || p.n * item % access != 0 || (p.m > 1 && p.ldy * item % access != 0))) access /= 2;
  if (access == 16) return run<T, 16>(op, p, how, st);
  if (access == 8) return run<T, 8>(op, p, how, st);
  if constexpr (sizeof(T) == 2) {
    if (access == 2) return run<T, 2>(op, p, how, st);
  }
  return run<T, 4>(op, p, how, st);
}

static bool too_large(int64_t m, int64_t n, int64_t k) { return m >= ckpt::kMaxRows || n > (1 << 17) || k > (1 << 17); }

}  // namespace wg
}  // namespace f2c

using namespace f2c;

extern "C" int64_t f2c_checkpoint_weight_grad_workspace(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || wg::too_large(m, n, k)) return 0;
  return wg::plan(m, n, k).bytes;
}

extern "C" int f2c_checkpoint_weight_grad(const void* dy, int64_t ldy, int dtype, const uint8_t* codes, int64_t ldq, const float* scales, int64_t m, int64_t n, int64_t k, void* dw,
                                          void* db, int flags, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "checkpoint_weight_grad";
  if (const int rc = ckpt::check_sizes(op, dtype, m, k)) return rc;
  F2C_REQUIRE(n >= 0, F2C_ERR_INVALID, "%s: negative size", op);
  F2C_REQUIRE(!wg::too_large(m, n, k), F2C_ERR_LIMIT, "%s: 2^31 rows, or more than 2^17 columns", op);
  F2C_REQUIRE((flags & ~F2C_NO_WAITS) == 0, F2C_ERR_INVALID, "%s: unknown flags", op);
  if (const int rc = ckpt::check_codes(op, codes, ldq, scales, m, k)) return rc;
  if (n == 0) return F2C_OK;
  F2C_REQUIRE(db && (dw || k == 0), F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(m == 0 || dy, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(m <= 1 || ldy >= n, F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  F2C_REQUIRE(k > 0 || m == 0, F2C_ERR_INVALID, "%s: no columns", op);
  cudaStream_t st = (cudaStream_t)stream;
  if (m == 0) {
    cudaError_t e = cudaMemsetAsync(db, 0, (size_t)(n * dtype_size(dtype)), st);
    if (e == cudaSuccess && k > 0) e = cudaMemsetAsync(dw, 0, (size_t)(n * k * dtype_size(dtype)), st);
    if (e != cudaSuccess) return set_error(F2C_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
    return F2C_OK;
  }
  const wg::Plan how = wg::plan(m, n, k);
  F2C_REQUIRE(how.bytes == 0 || (workspace && workspace_bytes >= how.bytes && aligned(workspace, 256)), F2C_ERR_INVALID,
              "%s: the workspace must have %lld bytes, 256-byte aligned", op, (long long)how.bytes);
  const wg::Params p{dy, ldy, m, (int)n, (int)k, ckpt::Codes{const_cast<uint8_t*>(codes), ldq, const_cast<float*>(scales), ceil_div(k, ckpt::kGroup)}, how.n_tiles, how.splits, how.split_rows,
               dw, db, (float*)workspace, (float*)((char*)workspace + how.part_bytes),
               (flags & F2C_NO_WAITS) ? 0u : t5::kWaitLimit, stream_error_word()};
  if (dtype == F2C_F32) return wg::run<float>(op, p, how, st);
  if (dtype == F2C_F16) return wg::run<__half>(op, p, how, st);
  return wg::run<__nv_bfloat16>(op, p, how, st);
}
