// Layer norm of rows, forward (f2c_layer_norm): y = (x - mean) rstd weight + bias, rstd = 1 / sqrt(mean((x - mean)^2) + eps), with or without
// ReLU; for training also mean, rstd, the ReLU's bits, and the rows in 8 bits (checkpoint.cuh), all of it in the one pass.
//
// Bound by reading and writing the rows.  A row's values stay in registers between the mean, the squares of the differences from it (no
// cancellation of large means) and the result: a warp has rows up to 1024 columns long, several at a time where they are short so that enough loads are on
// the way; a CTA has longer ones, and what its registers do not hold (beyond 16,384 columns) it reads again.
#include "checkpoint.cuh"

namespace f2c {
namespace ln {

using ckpt::Four;
using ckpt::kGroup;

struct Args {
  const void* x;
  int64_t ldx, m;
  int d;
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

// of four values of columns [at, at + 4) of a vector that starts anywhere
__device__ __forceinline__ void of_columns(const float* w, int at, int left, float otherwise, float (&v)[4]) {
  if (w == nullptr || left <= 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = otherwise;
  } else if (left >= 4 && (reinterpret_cast<uintptr_t>(w) & 15) == 0) {
    const float4 f = __ldg(reinterpret_cast<const float4*>(w + at));
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < left ? __ldg(w + at + e) : otherwise;
  }
}

// Everything that a lane writes of four columns of a row; by whole warps.
template <typename T, int ACCESS>
__device__ __forceinline__ void finish(const Args& a, int64_t row, int chunk, const float (&x)[4], float mean, float rstd, const float (&w)[4], const float (&b)[4]) {
  const int lane = threadIdx.x & 31, col = chunk * kGroup + 4 * lane, left = a.d - col;
  float z[4];
  uint32_t bits = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    z[e] = fmaf((x[e] - mean) * rstd, w[e], b[e]);
    if (e < left && z[e] > 0.0f) bits |= 1u << e;
    if (a.relu && z[e] < 0.0f) z[e] = 0.0f;  // (a NaN stays one)
  }
  Four<T, ACCESS> out;
  out.set(z);
  out.store((T*)a.y + row * a.d + col, left);
  if (a.active != nullptr) {
    bits |= __shfl_down_sync(0xffffffffu, bits, 1) << 4;
    if ((lane & 1) == 0 && left > 0) a.active[row * ((a.d + 7) >> 3) + (col >> 3)] = (uint8_t)bits;
  }
  if (a.codes.codes != nullptr) {
    ckpt::Scale s;
    const uint32_t q = ckpt::encode(x, left, s);
    if (left > 0) *reinterpret_cast<uint32_t*>(a.codes.codes + row * a.codes.ld + col) = q;
    if (lane == 0) ckpt::store_scale(a.codes.scales + 2 * (row * a.codes.groups + chunk), s);
  }
}

constexpr int kThreads = 256;

// ROWS rows of up to CHUNKS * 128 columns for every warp
template <typename T, int ACCESS, int CHUNKS, int ROWS>
__global__ void __launch_bounds__(kThreads) warp_kernel(const __grid_constant__ Args a) {
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t first = ((int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * ROWS;
  Four<T, ACCESS> raw[ROWS][CHUNKS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = c * kGroup + 4 * lane;
      raw[r][c].load((const T*)a.x + (first + r) * a.ldx + col, first + r < a.m ? a.d - col : 0);
    }
  float w[CHUNKS][4], b[CHUNKS][4];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int col = c * kGroup + 4 * lane;
    of_columns(a.weight, col, a.d - col, 1.0f, w[c]);
    of_columns(a.bias, col, a.d - col, 0.0f, b[c]);
  }
  const float n = (float)a.d;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t row = first + r;
    if (row >= a.m) return;  // all threads of the warp
    float x[CHUNKS][4], sum = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      raw[r][c].get(x[c]);
      sum += (x[c][0] + x[c][1]) + (x[c][2] + x[c][3]);
    }
    const float mean = warp_sum(sum) / n;
    float squares = 0.0f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float t = c * kGroup + 4 * lane + e < a.d ? x[c][e] - mean : 0.0f;
        squares = fmaf(t, t, squares);
      }
    const float rstd = 1.0f / sqrtf(warp_sum(squares) / n + a.eps);
    if (lane == 0 && a.mean != nullptr) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
      if (c * kGroup < a.d) finish<T, ACCESS>(a, row, c, x[c], mean, rstd, w[c], b[c]);
  }
}

template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float* of_warp) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) v += of_warp[w];
  return v;
}

// A row for every CTA: chunks warp, warp + THREADS / 32, ... are a warp's, KEPT of which it keeps.
template <typename T, int ACCESS, int THREADS, int KEPT>
__global__ void __launch_bounds__(THREADS) block_kernel(const __grid_constant__ Args a) {
  constexpr int kWarps = THREADS / 32;
  __shared__ float of_warp[2][kWarps];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, chunks = (a.d + kGroup - 1) / kGroup;
  const int64_t row = blockIdx.x;
  const T* const from = (const T*)a.x + row * a.ldx;
  Four<T, ACCESS> raw[KEPT];
#pragma unroll
  for (int k = 0; k < KEPT; ++k) {
    const int col = (warp + k * kWarps) * kGroup + 4 * lane;
    raw[k].load(from + col, a.d - col);
  }
  const auto each = [&](auto&& body) {  // every chunk of this warp
#pragma unroll
    for (int k = 0; k < KEPT; ++k) {
      if (warp + k * kWarps >= chunks) break;
      float x[4];
      raw[k].get(x);
      body(warp + k * kWarps, x);
    }
    for (int c = warp + KEPT * kWarps; c < chunks; c += kWarps) {
      Four<T, ACCESS> more;
      float x[4];
      const int col = c * kGroup + 4 * lane;
      more.load(from + col, a.d - col);
      more.get(x);
      body(c, x);
    }
  };
  const float n = (float)a.d;
  float sum = 0.0f;
  each([&](int, const float (&x)[4]) { sum += (x[0] + x[1]) + (x[2] + x[3]); });
  const float mean = block_sum<THREADS>(sum, of_warp[0]) / n;
  float squares = 0.0f;
  each([&](int c, const float (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float t = c * kGroup + 4 * lane + e < a.d ? x[e] - mean : 0.0f;
      squares = fmaf(t, t, squares);
    }
  });
  const float rstd = 1.0f / sqrtf(block_sum<THREADS>(squares, of_warp[1]) / n + a.eps);
  if (threadIdx.x == 0 && a.mean != nullptr) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  each([&](int c, const float (&x)[4]) {
    float w[4], b[4];
    const int col = c * kGroup + 4 * lane;
    of_columns(a.weight, col, a.d - col, 1.0f, w);
    of_columns(a.bias, col, a.d - col, 0.0f, b);
    finish<T, ACCESS>(a, row, c, x, mean, rstd, w, b);
  });
}

template <typename T, int ACCESS, int CHUNKS, int ROWS>
static void by_warps(const Args& a, cudaStream_t st) {
  launch_dependent(warp_kernel<T, ACCESS, CHUNKS, ROWS>, dim3((unsigned)ceil_div(a.m, kThreads / 32 * ROWS)), kThreads, 0, st, a);
}

template <typename T, int ACCESS>
static void run(const Args& a, cudaStream_t st) {
  if (a.d <= kGroup) by_warps<T, ACCESS, 1, 4>(a, st);
  else if (a.d <= 2 * kGroup) by_warps<T, ACCESS, 2, 2>(a, st);
  else if (a.d <= 4 * kGroup) by_warps<T, ACCESS, 4, 1>(a, st);
  else if (a.d <= 8 * kGroup) by_warps<T, ACCESS, 8, 1>(a, st);
  else if (a.d <= 32 * kGroup) launch_dependent(block_kernel<T, ACCESS, 256, 4>, dim3((unsigned)a.m), 256, 0, st, a);
  else launch_dependent(block_kernel<T, ACCESS, 512, 8>, dim3((unsigned)a.m), 512, 0, st, a);
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
  if (m == 0 || d == 0) return F2C_OK;
  F2C_REQUIRE(x && y, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(m == 1 || ldx >= d, F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  F2C_REQUIRE(m < ckpt::kMaxRows, F2C_ERR_LIMIT, "%s: 2^31 rows", op);
  const ln::Args a{x, ldx, m, (int)d, weight, bias, eps, relu, y, mean, rstd, active, ckpt::Codes{codes, ldq, scales, ceil_div(d, ckpt::kGroup)}};
  const int item = dtype_size(dtype), from = ckpt::access_of(x, ldx, m, d, item), to = ckpt::access_of(y, d, m, d, item);
  F2C_BY_ROWS(ln::run, dtype, (from < to ? from : to), a, (cudaStream_t)stream);
  return check_launch(op);
}
