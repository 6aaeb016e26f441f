// Layer norm of rows, forward (f2c_layer_norm): y = (x - mean) rstd weight + bias, rstd = 1 / sqrt(mean((x - mean)^2) + eps), with or without
// ReLU; for training also mean, rstd, the ReLU's bits, and the rows in 8 bits (checkpoint.cuh), all of it in the one pass.
//
// Bound by reading and writing the rows (16,384 x 4096 bfloat16: 53 us, 5.1 TB/s; 59,000 x 128 float32: 9.2 us, 6.6 TB/s, half of it from L2).  A row's values stay in registers
// between the mean, the differences from it and their squares, and the result.
//
// Large means.  The sum and its division by the columns lose some last places of the mean, which every difference then has too: rows of nothing but 1000.3 came out 0.02
// from their bias, with eps 1e-5, and rows of -3e4 +- 0.01 0.07.  The mean of the differences is what was lost: the result, the variance and the mean that is kept are
// corrected by it.  (8 % of the time: 48.2 and 8.3 us without.  Only for rows whose mean is large it took 51.8 and 8.8, and 32.6 instead of 32.0 with codes, 62,500 x 256
// float32: not worth results that depend on a limit.)  The mean that is kept is rounded to single precision, and the backward pass starts from it.
//
// A warp has rows up to 1024 columns long, several at a time where they are short so that enough loads are on the way; a CTA of four warps (eight beyond 4096 columns)
// has longer ones, one after the other, the next one's loads on the way: five or six of them to an SM (two of eight warps, their columns' weights in registers, waited more
// than they worked: 16,384 x 4096 bfloat16 64 us); rows beyond 8192 columns it reads again for every step (4000 x 16,384 bfloat16 116 us; with a few registers more, and one
// CTA less an SM, 135).
#include "checkpoint.cuh"

namespace f2c {
namespace ln {

using ckpt::both;
using ckpt::f32x2;
using ckpt::fma2;
using ckpt::Four;
using ckpt::kGroup;
using ckpt::mul2;
using ckpt::pair_of;
using ckpt::plus2;

struct Args {
  const void* x;
  int64_t ldx, m;
  int d;
  float per_column;            // 1 / d
  const float *weight, *bias;  // null: 1, 0
  float eps;
  int relu;
  void* y;                     // [m, d]
  float *mean, *rstd;          // null: not wanted
  uint8_t* active;             // null: not wanted; [m, (d + 7) / 8]
  ckpt::Codes codes;           // codes null: not wanted
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float2 warp_sum(float2 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return v;
}

// Four values of a vector, at `w` those of this lane's first columns (null: `otherwise`), where all four exist and start on 16 bytes
__device__ __forceinline__ void of_columns(const float* w, float otherwise, f32x2 (&v)[2]) {
  float4 f = make_float4(otherwise, otherwise, otherwise, otherwise);
  if (w != nullptr) f = __ldg(reinterpret_cast<const float4*>(w));
  v[0] = pair_of(f.x, f.y);
  v[1] = pair_of(f.z, f.w);
}
// the same of columns [at, at + 4) of a vector that starts anywhere.  (One by one in a function of its own: as a branch they were eight loads beside every two.)
static __device__ __noinline__ float4 one_by_one(const float* w, int left, float otherwise) {
  return make_float4(__ldg(w), left > 1 ? __ldg(w + 1) : otherwise, left > 2 ? __ldg(w + 2) : otherwise, left > 3 ? __ldg(w + 3) : otherwise);
}
__device__ __forceinline__ void of_columns(const float* w, int at, int left, float otherwise, f32x2 (&v)[2]) {
  float4 f = make_float4(otherwise, otherwise, otherwise, otherwise);
  if (w != nullptr && left > 0) {
    if (left >= 4 && (reinterpret_cast<uintptr_t>(w) & 15) == 0) f = __ldg(reinterpret_cast<const float4*>(w + at));
    else f = one_by_one(w + at, left, otherwise);
  }
  v[0] = pair_of(f.x, f.y);
  v[1] = pair_of(f.z, f.w);
}

// The differences from the mean and their squares, of the columns that there are.
struct Spread { f32x2 off = 0ull, squares = 0ull; };
__device__ __forceinline__ void add_spread(const f32x2 (&x)[2], f32x2 less, int left, Spread& sum) {
  f32x2 t[2] = {plus2(x[0], less), plus2(x[1], less)};
  if (left < 4) {
    t[0] = left > 1 ? t[0] : left > 0 ? pair_of(lo32(t[0]), 0.0f) : 0ull;
    t[1] = left > 2 ? pair_of(lo32(t[1]), 0.0f) : 0ull;
  }
  sum.off = plus2(plus2(sum.off, t[0]), t[1]);
  sum.squares = fma2(t[1], t[1], fma2(t[0], t[0], sum.squares));
}
// 1 / sqrt(v), a step of Newton's behind the instruction's two units in the last place.  (With __frsqrt_rn, and the sum divided by the columns: 60 us instead of 54 at 16,384 x 4096.)
__device__ __forceinline__ float rstd_of(float v) {
  const float r = rsqrtf(v), off = fmaf(-(v * r), r, 1.0f);
  return fabsf(off) < 1.0f ? fmaf(0.5f * r, off, r) : r;  // (v zero or infinite: as it is)
}
__device__ __forceinline__ float sum_of(f32x2 v) { return lo32(v) + hi32(v); }

// What a row's values are normalised by: the mean as the sum gave it, what it is off, and the reciprocal deviation.
struct Norm {
  float mean, off, rstd;
  // from the sums of the differences and of their squares
  __device__ __forceinline__ Norm(const Args& a, float mean, float2 sums) : mean(mean), off(sums.x * a.per_column) {
    const float variance = fmaf(-off, off, sums.y * a.per_column);
    rstd = rstd_of((variance < 0.0f ? 0.0f : variance) + a.eps);  // (a NaN stays one)
  }
  __device__ __forceinline__ void keep(const Args& a, int64_t row) const {
    a.mean[row] = mean + off;
    a.rstd[row] = rstd;
  }
};

// Everything that a lane writes of four columns of a row, of which `left` exist; by whole warps.
// KEEP: with what is wanted for the backward pass beside the result.
template <typename T, int ACCESS, bool KEEP>
__device__ __forceinline__ void finish(const Args& a, T* y, int64_t row, int chunk, int left, const f32x2 (&x)[2], const Norm& n, const f32x2 (&w)[2], const f32x2 (&b)[2]) {
  const int lane = threadIdx.x & 31, col = chunk * kGroup + 4 * lane;
  f32x2 z[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) z[h] = fma2(fma2(plus2(x[h], both(-n.mean)), both(n.rstd), both(-n.off * n.rstd)), w[h], b[h]);
  if (KEEP && a.active != nullptr) {
    uint32_t bits = (lo32(z[0]) > 0.0f) | (hi32(z[0]) > 0.0f) << 1 | (lo32(z[1]) > 0.0f) << 2 | (hi32(z[1]) > 0.0f) << 3;
    if (left < 4) bits &= (1u << max(left, 0)) - 1u;
    bits |= __shfl_down_sync(0xffffffffu, bits, 1) << 4;
    if ((lane & 1) == 0 && left > 0) a.active[row * ((a.d + 7) >> 3) + (col >> 3)] = (uint8_t)bits;
  }
  if (a.relu) {  // (a NaN stays one)
#pragma unroll
    for (int h = 0; h < 2; ++h) z[h] = pair_of(ckpt::max_nan(lo32(z[h]), 0.0f), ckpt::max_nan(hi32(z[h]), 0.0f));
  }
  Four<T, ACCESS> out;
  out.set(z);
  out.store(y, left);
  if (KEEP && a.codes.codes != nullptr) {
    ckpt::Scale s;
    const uint32_t q = ckpt::encode(x, left, s);
    if (left > 0) *reinterpret_cast<uint32_t*>(a.codes.codes + row * a.codes.ld + col) = q;
    if (lane == 0) ckpt::store_scale(a.codes.scales + 2 * (row * a.codes.groups + chunk), s);
  }
}

constexpr int kThreads = 256;

// ROWS rows of CHUNKS * 128 columns for every warp; the last chunk may have fewer, unless EVEN.  (Four CTAs an SM up to 640 columns, three beyond, though a few registers
// spill: 16 M values with their codes, 256 columns 28 us and 31 with three, 768 columns 29 and 35 with two.)
template <typename T, int ACCESS, int CHUNKS, int ROWS, bool EVEN, bool KEEP>
__global__ void __launch_bounds__(kThreads, CHUNKS <= 5 ? 4 : 3) warp_kernel(const __grid_constant__ Args a) {
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t first = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * ROWS;
  const auto left_of = [&](int c) { return EVEN || c + 1 < CHUNKS ? 4 : a.d - c * kGroup - 4 * lane; };
  Four<T, ACCESS> raw[ROWS][CHUNKS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const T* const x = (const T*)a.x + (first + r) * a.ldx + 4 * lane;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) raw[r][c].load(x + c * kGroup, first + r < a.m ? left_of(c) : 0);
  }
  constexpr int kHeld = ROWS > 1 ? CHUNKS : 1;  // of weights: all where they are used more than once, or the first chunk's
  f32x2 w[kHeld][2], b[kHeld][2];
  const float *const weight = EVEN && a.weight != nullptr ? a.weight + 4 * lane : a.weight, *const bias = EVEN && a.bias != nullptr ? a.bias + 4 * lane : a.bias;
  const auto weights = [&](int c, f32x2 (&w)[2], f32x2 (&b)[2]) {
    if constexpr (EVEN) {
      of_columns(weight != nullptr ? weight + c * kGroup : nullptr, 1.0f, w);
      of_columns(bias != nullptr ? bias + c * kGroup : nullptr, 0.0f, b);
    } else {
      of_columns(weight, c * kGroup + 4 * lane, left_of(c), 1.0f, w);
      of_columns(bias, c * kGroup + 4 * lane, left_of(c), 0.0f, b);
    }
  };
#pragma unroll
  for (int c = 0; c < kHeld; ++c) weights(c, w[c], b[c]);
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t row = first + r;
    if (row >= a.m) return;  // all threads of the warp
    f32x2 x[CHUNKS][2], sum = 0ull;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      raw[r][c].get(x[c]);
      sum = plus2(plus2(sum, x[c][0]), x[c][1]);
    }
    const float mean = warp_sum(sum_of(sum)) * a.per_column;
    Spread spread;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) add_spread(x[c], both(-mean), left_of(c), spread);
    const Norm n(a, mean, warp_sum(make_float2(sum_of(spread.off), sum_of(spread.squares))));
    if (KEEP && lane == 0 && a.mean != nullptr) n.keep(a, row);
    T* const y = (T*)a.y + row * a.d + 4 * lane;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      if constexpr (ROWS > 1) {
        finish<T, ACCESS, KEEP>(a, y + c * kGroup, row, c, left_of(c), x[c], n, w[c], b[c]);
      } else {  // the next chunk's weights are on the way meanwhile
        f32x2 w_next[2], b_next[2];
        if (c + 1 < CHUNKS) weights(c + 1, w_next, b_next);
        finish<T, ACCESS, KEEP>(a, y + c * kGroup, row, c, left_of(c), x[c], n, w[0], b[0]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          w[0][h] = w_next[h];
          b[0][h] = b_next[h];
        }
      }
    }
  }
}

template <int THREADS, typename V>  // float or float2
__device__ __forceinline__ V block_sum(V v, V* of_warp) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = of_warp[threadIdx.x & (THREADS / 32 - 1)];
#pragma unroll
  for (int o = THREADS / 64; o > 0; o >>= 1) {
    if constexpr (sizeof(V) == sizeof(float)) {
      v += __shfl_xor_sync(0xffffffffu, v, o);
    } else {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
  }
  return v;
}

// A CTA has every gridDim.x-th row: chunks warp, warp + THREADS / 32, ... are a warp's, all of which it keeps.
template <typename T, int ACCESS, int THREADS, int KEPT, bool EVEN, bool KEEP>
__global__ void __launch_bounds__(THREADS, (KEEP ? 640 : 768) / THREADS) block_kernel(const __grid_constant__ Args a) {
  constexpr int kWarps = THREADS / 32;
  __shared__ float sums[kWarps];
  __shared__ float2 spreads[kWarps];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Four<T, ACCESS> next[KEPT];
  const int own = warp * kGroup + 4 * lane;  // this lane's first columns
  const auto fetch = [&](int64_t row) {
    const T* const x = (const T*)a.x + row * a.ldx + own;
    const int left = row < a.m ? a.d - own : 0;
#pragma unroll
    for (int k = 0; k < KEPT; ++k) next[k].load(x + k * (kWarps * kGroup), left - k * (kWarps * kGroup));
  };
  const int mine = max(0, min(KEPT, ((a.d + kGroup - 1) / kGroup - warp + kWarps - 1) / kWarps));  // chunks that there are
  fetch(blockIdx.x);
  for (int64_t row = blockIdx.x; row < a.m; row += gridDim.x) {
    f32x2 x[KEPT][2], sum = 0ull;
    Spread spread;
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
      next[k].get(x[k]);
      sum = plus2(plus2(sum, x[k][0]), x[k][1]);
    }
    fetch(row + gridDim.x);
    // (the barrier of one sum keeps the reads of the other's apart from the next row's writes)
    const float mean = block_sum<THREADS>(sum_of(sum), sums) * a.per_column;
#pragma unroll
    for (int k = 0; k < KEPT; ++k)
      if (k < mine) add_spread(x[k], both(-mean), EVEN ? 4 : a.d - (warp + k * kWarps) * kGroup - 4 * lane, spread);
    const Norm n(a, mean, block_sum<THREADS>(make_float2(sum_of(spread.off), sum_of(spread.squares)), spreads));
    if (KEEP && threadIdx.x == 0 && a.mean != nullptr) n.keep(a, row);
    T* const y = (T*)a.y + row * a.d + own;
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
      if (k >= mine) break;
      constexpr int kStep = kWarps * kGroup;
      const int left = EVEN ? 4 : a.d - own - k * kStep;
      f32x2 w[2], b[2];
      if constexpr (EVEN) {
        of_columns(a.weight != nullptr ? a.weight + own + k * kStep : nullptr, 1.0f, w);
        of_columns(a.bias != nullptr ? a.bias + own + k * kStep : nullptr, 0.0f, b);
      } else {
        of_columns(a.weight, own + k * kStep, left, 1.0f, w);
        of_columns(a.bias, own + k * kStep, left, 0.0f, b);
      }
      finish<T, ACCESS, KEEP>(a, y + k * kStep, row, warp + k * kWarps, left, x[k], n, w, b);
    }
  }
}

// Longer rows, one a CTA, read three times.
template <typename T, int ACCESS, bool KEEP>
__global__ void __launch_bounds__(512, KEEP ? 3 : 4) long_kernel(const __grid_constant__ Args a) {
  constexpr int kWarps = 16;
  __shared__ float sums[kWarps];
  __shared__ float2 spreads[kWarps];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, chunks = (a.d + kGroup - 1) / kGroup;
  const int64_t row = blockIdx.x;
  const T* const from = (const T*)a.x + row * a.ldx;
  const auto each = [&](auto&& body) {  // every chunk of this warp
#pragma unroll 4
    for (int c = warp; c < chunks; c += kWarps) {
      Four<T, ACCESS> v;
      f32x2 x[2];
      const int col = c * kGroup + 4 * lane;
      v.load(from + col, a.d - col);
      v.get(x);
      body(c, col, x);
    }
  };
  f32x2 sum = 0ull;
  Spread spread;
  each([&](int, int, const f32x2 (&x)[2]) { sum = plus2(plus2(sum, x[0]), x[1]); });
  const float mean = block_sum<512>(sum_of(sum), sums) * a.per_column;
  each([&](int, int col, const f32x2 (&x)[2]) { add_spread(x, both(-mean), a.d - col, spread); });
  const Norm n(a, mean, block_sum<512>(make_float2(sum_of(spread.off), sum_of(spread.squares)), spreads));
  if (KEEP && threadIdx.x == 0 && a.mean != nullptr) n.keep(a, row);
  each([&](int c, int col, const f32x2 (&x)[2]) {
    f32x2 w[2], b[2];
    of_columns(a.weight, col, a.d - col, 1.0f, w);
    of_columns(a.bias, col, a.d - col, 0.0f, b);
    finish<T, ACCESS, KEEP>(a, (T*)a.y + row * a.d + col, row, c, a.d - col, x, n, w, b);
  });
}

template <typename T, int ACCESS, int CHUNKS, int ROWS, bool EVEN, bool KEEP>
static void by_warps(const Args& a, cudaStream_t st) {
  launch_dependent(warp_kernel<T, ACCESS, CHUNKS, ROWS, EVEN, KEEP>, dim3((unsigned)ceil_div(a.m, kThreads / 32 * ROWS)), kThreads, 0, st, a);
}
template <typename T, int ACCESS, int THREADS, int KEPT, bool EVEN, bool KEEP>
static void by_ctas(const Args& a, int resident, cudaStream_t st) {
  const int64_t most = (int64_t)resident * kSmCount;
  launch_dependent(block_kernel<T, ACCESS, THREADS, KEPT, EVEN, KEEP>, dim3((unsigned)(a.m < most ? a.m : most)), THREADS, 0, st, a);
}

template <typename T, int ACCESS, bool EVEN, bool KEEP>
static void by_size(const Args& a, cudaStream_t st) {
  switch ((a.d + kGroup - 1) / kGroup) {
    case 1: return by_warps<T, ACCESS, 1, 4, EVEN, KEEP>(a, st);
    case 2: return by_warps<T, ACCESS, 2, 2, EVEN, KEEP>(a, st);
    case 3: return by_warps<T, ACCESS, 3, 1, EVEN, KEEP>(a, st);
    case 4: return by_warps<T, ACCESS, 4, 1, EVEN, KEEP>(a, st);
    case 5: return by_warps<T, ACCESS, 5, 1, EVEN, KEEP>(a, st);
    case 6: return by_warps<T, ACCESS, 6, 1, EVEN, KEEP>(a, st);
    case 7: return by_warps<T, ACCESS, 7, 1, EVEN, KEEP>(a, st);
    case 8: return by_warps<T, ACCESS, 8, 1, EVEN, KEEP>(a, st);
    default: break;
  }
  if (a.d <= 16 * kGroup) by_ctas<T, ACCESS, 128, 4, EVEN, KEEP>(a, KEEP ? 5 : 6, st);
  else if (a.d <= 32 * kGroup) by_ctas<T, ACCESS, 128, 8, EVEN, KEEP>(a, KEEP ? 5 : 6, st);
  else if (a.d <= 64 * kGroup) by_ctas<T, ACCESS, 256, 8, EVEN, KEEP>(a, KEEP ? 2 : 3, st);
  else launch_dependent(long_kernel<T, ACCESS, KEEP>, dim3((unsigned)a.m), 512, 0, st, a);
}
template <typename T, int ACCESS>
static void run(const Args& a, cudaStream_t st) {
  const bool keep = a.mean != nullptr || a.active != nullptr || a.codes.codes != nullptr;
  if constexpr (ACCESS == 4 * (int)sizeof(T)) {
    if (a.d % kGroup == 0 && aligned(a.weight, 16) && aligned(a.bias, 16)) return keep ? by_size<T, ACCESS, true, true>(a, st) : by_size<T, ACCESS, true, false>(a, st);
  }
  keep ? by_size<T, ACCESS, false, true>(a, st) : by_size<T, ACCESS, false, false>(a, st);
}

}  // namespace ln
}  // namespace f2c

using namespace f2c;

extern "C" int f2c_layer_norm(const void* x, int64_t ldx, int dtype, int64_t m, int64_t d, const float* weight, const float* bias, float eps, int relu, void* y,
                              float* mean, float* rstd, uint8_t* active, uint8_t* codes, int64_t ldq, float* scales, void* stream) {
  const char* op = "layer_norm";
  if (const int rc = ckpt::check_sizes(op, dtype, m, d)) return rc;
  F2C_REQUIRE(eps >= 0.0f, F2C_ERR_INVALID, "%s: eps must not be negative", op);  // (nor a NaN)
  F2C_REQUIRE((mean == nullptr) == (rstd == nullptr), F2C_ERR_INVALID, "%s: mean and rstd go together", op);
  if (codes || scales)
    if (const int rc = ckpt::check_codes(op, codes, ldq, scales, m, d)) return rc;
  if (m > 0 && d == 0 && mean != nullptr) {  // the mean of no values
    cudaError_t e = cudaMemsetAsync(mean, 0xff, (size_t)m * sizeof(float), (cudaStream_t)stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(rstd, 0xff, (size_t)m * sizeof(float), (cudaStream_t)stream);
    if (e != cudaSuccess) return set_error(F2C_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
  }
  if (m == 0 || d == 0) return F2C_OK;
  F2C_REQUIRE(x && y, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(m == 1 || ldx >= d, F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  F2C_REQUIRE(m < ckpt::kMaxRows, F2C_ERR_LIMIT, "%s: 2^31 rows", op);
  const ln::Args a{x, ldx, m, (int)d, (float)(1.0 / (double)d), weight, bias, eps, relu, y, mean, rstd, active, ckpt::Codes{codes, ldq, scales, ceil_div(d, ckpt::kGroup)}};
  const int item = dtype_size(dtype), from = ckpt::access_of(x, ldx, m, d, item), to = ckpt::access_of(y, d, m, d, item);
  F2C_BY_ROWS(ln::run, dtype, (from < to ? from : to), a, (cudaStream_t)stream);
  return check_launch(op);
}
