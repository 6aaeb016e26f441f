// Layer norm's backward pass (f2c_layer_norm_backward).  With h = (x - mean) rstd and g = dy where the ReLU was open (everywhere without one):
//   dx = rstd (g w - mean(g w) - h mean(g w h)),   dweight = sum over rows of g h,   dbias = sum over rows of g.
// x is the rows themselves or their 8-bit codes (checkpoint.cuh), decoded on the way.
//
// Bound by reading dy and x and writing dx (59,000 x 128 float32: 15 us, 6.0 TB/s; 37,237 x 256 from 8 bits with the ReLU's bits: 18 us, 4.8 TB/s; the launch
// that joins the sums 2 to 4 us).  A lane has the same columns of every row that its warp (or CTA) takes, so the sums over rows stay in
// registers; each CTA leaves one part of them, and a second launch adds the parts up in their order: no atomics, the same bits every time.
// What a row needs is on the way while the row before it is worked on.
#include <type_traits>

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

struct Back {
  const void* dy;
  int64_t ldy;
  const void* x;               // or
  ckpt::Codes codes;
  int64_t ldx, m;
  int d;
  float per_column;            // 1 / d
  const float *mean, *rstd;
  const uint8_t* active;       // null: no ReLU
  const float* weight;         // null: 1
  void* dx;                    // [m, d]
  float *dw, *db;              // a CTA's sums, those of the next one `part` further: [CTAs][2][d], or the results where there is one CTA
  int64_t part;
};

// A lane's four columns of a row, on their way
template <typename T, int ACCESS, bool CODES>
struct Columns {
  using Kept = typename std::conditional<CODES, uint32_t, Four<T, ACCESS>>::type;
  Four<T, ACCESS> dy;
  Kept x;
  ckpt::Scale s;
  uint32_t open;

  // `at`: the row, from this lane's columns of its first chunk on; this chunk's are `step` columns further, of which `left` exist (none: nothing is loaded)
  struct Row {
    const T *dy, *x;
    const uint8_t *codes, *active;
    const float* scales;
    __device__ __forceinline__ Row(const Back& a, int64_t row, int member) {
      const int own = member * kGroup + 4 * (threadIdx.x & 31);
      dy = (const T*)a.dy + row * a.ldy + own;
      if constexpr (CODES) {
        codes = a.codes.codes + row * a.codes.ld + own;
        scales = a.codes.scales + 2 * (row * a.codes.groups + member);
      } else {
        x = (const T*)a.x + row * a.ldx + own;
      }
      active = a.active + row * ((a.d + 7) >> 3) + (own >> 3);
    }
  };
  __device__ __forceinline__ void load(const Row& at, int step, int left, bool masked) {
    dy.load(at.dy + step, left);
    if constexpr (CODES) {
      x = ldg_nc_u32_if(at.codes + step, left > 0);
      const uint2 v = ckpt::ld_u64_if(at.scales + 2 * (step / kGroup), left > 0);
      s = ckpt::Scale{__uint_as_float(v.x), __uint_as_float(v.y)};
    } else {
      x.load(at.x + step, left);
    }
    open = masked && left > 0 ? (uint32_t)__ldg(at.active + (step >> 3)) >> (4 * (threadIdx.x & 1)) : 15u;
  }
  // g and h; columns that do not exist have no g (what they have for h meets nothing else)
  __device__ __forceinline__ void get(bool masked, float mean, float rstd, f32x2 (&g)[2], f32x2 (&h)[2]) const {
    dy.get(g);
    if (masked) {
      g[0] = pair_of(open & 1u ? lo32(g[0]) : 0.0f, open & 2u ? hi32(g[0]) : 0.0f);
      g[1] = pair_of(open & 4u ? lo32(g[1]) : 0.0f, open & 8u ? hi32(g[1]) : 0.0f);
    }
    if constexpr (CODES) ckpt::decode(x, s, h);
    else x.get(h);
#pragma unroll
    for (int q = 0; q < 2; ++q) h[q] = mul2(plus2(h[q], both(-mean)), both(rstd));
  }
};

__device__ __forceinline__ void weights_of(const Back& a, int chunk, f32x2 (&w)[2]) {
  const int col = chunk * kGroup + 4 * (threadIdx.x & 31);
  float f[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = col + e < a.d ? (a.weight != nullptr ? __ldg(a.weight + col + e) : 1.0f) : 0.0f;
  w[0] = pair_of(f[0], f[1]);
  w[1] = pair_of(f[2], f[3]);
}

__device__ __forceinline__ void warp_sum2(float& u, float& v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    u += __shfl_xor_sync(0xffffffffu, u, o);
    v += __shfl_xor_sync(0xffffffffu, v, o);
  }
}

// WARPS warps have a row of up to WARPS * CHUNKS * 128 columns: one warp, two, or all of a CTA.
template <typename T, int ACCESS, bool CODES, int WARPS, int CHUNKS, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 512 ? 1 : CHUNKS == 1 ? 3 : 2) backward_kernel(const __grid_constant__ Back a) {
  constexpr int kRows = THREADS / 32 / WARPS;  // of a CTA at a time
  constexpr bool kAlone = WARPS == 1;
  constexpr int kColumns = WARPS * CHUNKS * kGroup;
  __shared__ float sums[2][2][kAlone ? 1 : THREADS / 32];
  __shared__ float joined[kRows > 1 ? 2 * kColumns : 1][kRows > 1 ? kRows + 1 : 1];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, member = warp % WARPS, own = warp / WARPS * WARPS;
  const int64_t stride = (int64_t)gridDim.x * kRows;
  int64_t row = (int64_t)blockIdx.x * kRows + warp / WARPS;
  Columns<T, ACCESS, CODES> next[CHUNKS];
  float next_mean = 0.0f, next_rstd = 0.0f;
  const bool masked = a.active != nullptr;
  const auto fetch = [&](int64_t r) {
    if (r >= a.m) return;
    const typename Columns<T, ACCESS, CODES>::Row at(a, r, member);
    const int left = a.d - member * kGroup - 4 * lane;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) next[c].load(at, c * WARPS * kGroup, left - c * WARPS * kGroup, masked);
    next_mean = __ldg(a.mean + r);
    next_rstd = __ldg(a.rstd + r);
  };
  fetch(row);
  constexpr bool kHeld = WARPS < 16;  // (the widest rows' weights do not fit beside their sums: they are read again for every row)
  f32x2 held[kHeld ? CHUNKS : 1][2], dw[CHUNKS][2], db[CHUNKS][2];
  const auto weights = [&](int c, f32x2 (&w)[2]) {
    if constexpr (kHeld) {
#pragma unroll
      for (int q = 0; q < 2; ++q) w[q] = held[c][q];
    } else {
      weights_of(a, member + c * WARPS, w);
    }
  };
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    if constexpr (kHeld) weights_of(a, member + c * WARPS, held[c]);
#pragma unroll
    for (int q = 0; q < 2; ++q) dw[c][q] = db[c][q] = 0ull;
  }
  // (all warps of a row leave together)
  for (int turn = 0; row < a.m; row += stride, turn ^= 1) {
    const float rstd = next_rstd;
    f32x2 g[CHUNKS][2], h[CHUNKS][2];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) next[c].get(masked, next_mean, rstd, g[c], h[c]);
    fetch(row + stride);
    f32x2 us = 0ull, vs = 0ull;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      f32x2 w[2];
      weights(c, w);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        dw[c][q] = fma2(g[c][q], h[c][q], dw[c][q]);
        db[c][q] = plus2(db[c][q], g[c][q]);
        g[c][q] = mul2(g[c][q], w[q]);
        us = plus2(us, g[c][q]);
        vs = fma2(g[c][q], h[c][q], vs);
      }
    }
    float u = lo32(us) + hi32(us), v = lo32(vs) + hi32(vs);
    warp_sum2(u, v);
    if constexpr (!kAlone) {
      if (lane == 0) {
        sums[turn][0][warp] = u;
        sums[turn][1][warp] = v;
      }
      // of the row's warps (the other turn's sums are read before the next one)
      if constexpr (kRows == 1) __syncthreads();
      else asm volatile("bar.sync %0, %1;" ::"r"(warp / WARPS + 1), "n"(WARPS * 32) : "memory");
      u = v = 0.0f;
#pragma unroll
      for (int q = 0; q < WARPS; ++q) {
        u += sums[turn][0][own + q];
        v += sums[turn][1][own + q];
      }
    }
    u *= a.per_column;
    v *= a.per_column;
    T* const dx = (T*)a.dx + row * a.d + member * kGroup + 4 * lane;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      constexpr int kStep = WARPS * kGroup;
#pragma unroll
      for (int q = 0; q < 2; ++q) g[c][q] = mul2(both(rstd), fma2(h[c][q], both(-v), plus2(g[c][q], both(-u))));
      Four<T, ACCESS> out;
      out.set(g[c]);
      out.store(dx + c * kStep, a.d - member * kGroup - 4 * lane - c * kStep);
    }
  }
  float *const part_dw = a.dw + blockIdx.x * a.part, *const part_db = a.db + blockIdx.x * a.part;
  if constexpr (kRows > 1) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int col = (member + c * WARPS) * kGroup + 4 * lane + e;
        joined[col][warp / WARPS] = e & 1 ? hi32(dw[c][e / 2]) : lo32(dw[c][e / 2]);
        joined[kColumns + col][warp / WARPS] = e & 1 ? hi32(db[c][e / 2]) : lo32(db[c][e / 2]);
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.d; i += THREADS) {
      const int from = i < a.d ? i : kColumns + i - a.d;
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < kRows; ++q) sum += joined[from][q];
      if (i < a.d) part_dw[i] = sum;
      else part_db[i - a.d] = sum;
    }
  } else {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int col = (member + c * WARPS) * kGroup + 4 * lane;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col + e < a.d) {
          part_dw[col + e] = e & 1 ? hi32(dw[c][e / 2]) : lo32(dw[c][e / 2]);
          part_db[col + e] = e & 1 ? hi32(db[c][e / 2]) : lo32(db[c][e / 2]);
        }
    }
  }
}

// Rows that a CTA's registers do not hold: dx alone, each row read twice; the sums over rows are columns_kernel's.
template <typename T, int ACCESS, bool CODES>
__global__ void __launch_bounds__(512) long_kernel(const __grid_constant__ Back a) {
  constexpr int kWarps = 16;
  __shared__ float sums[2][kWarps];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, chunks = (a.d + kGroup - 1) / kGroup;
  const int64_t row = blockIdx.x;
  const float mean = __ldg(a.mean + row), rstd = __ldg(a.rstd + row);
  const typename Columns<T, ACCESS, CODES>::Row at(a, row, 0);
  float u = 0.0f, v = 0.0f;
  f32x2 us = 0ull, vs = 0ull;
  for (int pass = 0; pass < 2; ++pass) {
    for (int c = warp; c < chunks; c += kWarps) {
      Columns<T, ACCESS, CODES> now;
      f32x2 g[2], h[2], w[2];
      const int col = c * kGroup + 4 * lane, left = a.d - col;
      now.load(at, c * kGroup, left, a.active != nullptr);
      now.get(a.active != nullptr, mean, rstd, g, h);
      weights_of(a, c, w);
      if (pass == 0) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const f32x2 gw = mul2(g[q], w[q]);
          us = plus2(us, gw);
          vs = fma2(gw, h[q], vs);
        }
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) g[q] = mul2(both(rstd), fma2(h[q], both(-v), fma2(g[q], w[q], both(-u))));
        Four<T, ACCESS> out;
        out.set(g);
        out.store((T*)a.dx + row * a.d + col, left);
      }
    }
    if (pass == 0) {
      u = lo32(us) + hi32(us);
      v = lo32(vs) + hi32(vs);
      warp_sum2(u, v);
      if (lane == 0) {
        sums[0][warp] = u;
        sums[1][warp] = v;
      }
      __syncthreads();
      u = v = 0.0f;
#pragma unroll
      for (int q = 0; q < kWarps; ++q) {
        u += sums[0][q];
        v += sums[1][q];
      }
      u *= a.per_column;
      v *= a.per_column;
    }
  }
}

// The sums of such rows: a CTA has 128 columns of every gridDim.x-th stretch of eight rows.
template <typename T, int ACCESS, bool CODES>
__global__ void __launch_bounds__(256) columns_kernel(const __grid_constant__ Back a) {
  __shared__ float joined[2 * kGroup][9];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  f32x2 dw[2] = {}, db[2] = {};
  for (int64_t row = (int64_t)blockIdx.x * 8 + warp; row < a.m; row += (int64_t)gridDim.x * 8) {
    Columns<T, ACCESS, CODES> now;
    now.load(typename Columns<T, ACCESS, CODES>::Row(a, row, blockIdx.y), 0, a.d - (int)blockIdx.y * kGroup - 4 * lane, a.active != nullptr);
    f32x2 g[2], h[2];
    now.get(a.active != nullptr, __ldg(a.mean + row), __ldg(a.rstd + row), g, h);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      dw[q] = fma2(g[q], h[q], dw[q]);
      db[q] = plus2(db[q], g[q]);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    joined[4 * lane + e][warp] = e & 1 ? hi32(dw[e / 2]) : lo32(dw[e / 2]);
    joined[kGroup + 4 * lane + e][warp] = e & 1 ? hi32(db[e / 2]) : lo32(db[e / 2]);
  }
  __syncthreads();
  const int which = threadIdx.x / kGroup, c = threadIdx.x % kGroup, at = blockIdx.y * kGroup + c;
  float sum = 0.0f;
#pragma unroll
  for (int q = 0; q < 8; ++q) sum += joined[which * kGroup + c][q];
  if (at < a.d) (which ? a.db : a.dw)[blockIdx.x * a.part + at] = sum;
}

// The parts' sums: eight columns a CTA, four parts a warp at a time, a warp for every 16 parts.  (32 columns a CTA and a part a warp took 8 us for 888 parts of 256.)
__global__ void __launch_bounds__(1024) join_kernel(const float* __restrict__ parts, int count, int d, float* __restrict__ dweight, float* __restrict__ dbias) {
  __shared__ float of[32][8];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, at = blockIdx.x * 8 + (lane & 7);
  float sum = 0.0f;
  if (at < 2 * d) {
#pragma unroll 8
    for (int p = warp * 4 + (lane >> 3); p < count; p += 4 * warps) sum += parts[(int64_t)p * 2 * d + at];
  }
  sum += __shfl_xor_sync(0xffffffffu, sum, 8);
  sum += __shfl_xor_sync(0xffffffffu, sum, 16);
  if (lane < 8) of[warp][lane] = sum;
  __syncthreads();
  if (threadIdx.x >= 8) return;
  sum = 0.0f;
  for (int q = 0; q < warps; ++q) sum += of[q][lane];
  if (at < d) {
    if (dweight != nullptr) dweight[at] = sum;
  } else if (at < 2 * d && dbias != nullptr) {
    dbias[at - d] = sum;
  }
}

// How the rows are dealt out: columns that a CTA's registers hold, and CTAs.  (Three chunks by themselves: 384 columns of 16 M float32 values 34 us, and 41 as four.)
struct Deal {
  int warps, chunks, threads;  // warps 0: too long
  int ctas;
};
static Deal deal(int64_t m, int64_t d) {
  Deal r;
  if (d <= kGroup) r = {1, 1, 256, 3};
  else if (d <= 2 * kGroup) r = {1, 2, 256, 2};
  else if (d <= 3 * kGroup) r = {1, 3, 256, 2};
  else if (d <= 4 * kGroup) r = {1, 4, 256, 2};
  else if (d <= 6 * kGroup) r = {2, 3, 256, 2};
  else if (d <= 8 * kGroup) r = {2, 4, 256, 2};
  else if (d <= 16 * kGroup) r = {8, 2, 256, 2};
  else if (d <= 32 * kGroup) r = {8, 4, 256, 2};
  else if (d <= 64 * kGroup) r = {16, 4, 512, 1};
  else r = {0, 1, 256, 1};
  const int rows = r.warps == 0 ? 8 : r.threads / 32 / r.warps;
  int64_t ctas = ceil_div(m, rows), most = (int64_t)kSmCount * r.ctas;  // (a constant: results do not depend on the device's count)
  if (r.warps == 0) most = 64;
  r.ctas = (int)(ctas < most ? ctas : most);
  return r;
}

template <typename T, int ACCESS, bool CODES>
static void run_source(const Back& a, const Deal& how, cudaStream_t st) {
  const dim3 grid((unsigned)how.ctas);
  if (how.warps == 1 && how.chunks == 1) launch_dependent(backward_kernel<T, ACCESS, CODES, 1, 1, 256>, grid, 256, 0, st, a);
  else if (how.warps == 1 && how.chunks == 2) launch_dependent(backward_kernel<T, ACCESS, CODES, 1, 2, 256>, grid, 256, 0, st, a);
  else if (how.warps == 1 && how.chunks == 3) launch_dependent(backward_kernel<T, ACCESS, CODES, 1, 3, 256>, grid, 256, 0, st, a);
  else if (how.warps == 1) launch_dependent(backward_kernel<T, ACCESS, CODES, 1, 4, 256>, grid, 256, 0, st, a);
  else if (how.warps == 2 && how.chunks == 3) launch_dependent(backward_kernel<T, ACCESS, CODES, 2, 3, 256>, grid, 256, 0, st, a);
  else if (how.warps == 2) launch_dependent(backward_kernel<T, ACCESS, CODES, 2, 4, 256>, grid, 256, 0, st, a);
  else if (how.warps == 8 && how.chunks == 2) launch_dependent(backward_kernel<T, ACCESS, CODES, 8, 2, 256>, grid, 256, 0, st, a);
  else if (how.warps == 8) launch_dependent(backward_kernel<T, ACCESS, CODES, 8, 4, 256>, grid, 256, 0, st, a);
  else if (how.warps == 16) launch_dependent(backward_kernel<T, ACCESS, CODES, 16, 4, 512>, grid, 512, 0, st, a);
  else {
    launch_dependent(long_kernel<T, ACCESS, CODES>, dim3((unsigned)a.m), 512, 0, st, a);
    launch_dependent(columns_kernel<T, ACCESS, CODES>, dim3((unsigned)how.ctas, (unsigned)ceil_div(a.d, kGroup)), 256, 0, st, a);
  }
}
template <typename T, int ACCESS>
static void run(const Back& a, const Deal& how, cudaStream_t st) {
  if (a.codes.codes != nullptr) run_source<T, ACCESS, true>(a, how, st);
  else run_source<T, ACCESS, false>(a, how, st);
}

}  // namespace ln
}  // namespace f2c

using namespace f2c;

extern "C" int64_t f2c_layer_norm_backward_workspace(int64_t m, int64_t d) {
  if (m <= 0 || d <= 0 || m >= ckpt::kMaxRows || d > ckpt::kMaxColumns) return 0;
  return ceil_div((int64_t)ln::deal(m, d).ctas * 2 * d * 4, 256) * 256;
}

extern "C" int f2c_layer_norm_backward(const void* dy, int64_t ldy, int dtype, const void* x, int64_t ldx, const uint8_t* codes, int64_t ldq, const float* scales,
                                       const float* mean, const float* rstd, const uint8_t* active, const float* weight, int64_t m, int64_t d, void* dx,
                                       float* dweight, float* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "layer_norm_backward";
  if (const int rc = ckpt::check_sizes(op, dtype, m, d)) return rc;
  F2C_REQUIRE(x == nullptr || codes == nullptr, F2C_ERR_INVALID, "%s: rows or their codes, not both", op);
  if (codes || scales)
    if (const int rc = ckpt::check_codes(op, codes, ldq, scales, m, d)) return rc;
  if (d == 0) return F2C_OK;
  F2C_REQUIRE(m == 0 || ((x || codes) && dy && mean && rstd && dx), F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(m <= 1 || (ldy >= d && (x == nullptr || ldx >= d)), F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  F2C_REQUIRE(m < ckpt::kMaxRows, F2C_ERR_LIMIT, "%s: 2^31 rows", op);
  const int64_t need = f2c_layer_norm_backward_workspace(m, d);
  F2C_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 256)), F2C_ERR_INVALID, "%s: the workspace must have %lld bytes, 256-byte aligned", op,
              (long long)need);
  cudaStream_t st = (cudaStream_t)stream;
  const ln::Deal how = ln::deal(m, d);
  const bool alone = m > 0 && how.ctas == 1 && dweight != nullptr && dbias != nullptr;  // nothing to join
  if (m > 0) {
    const ln::Back a{dy, ldy, x, ckpt::Codes{const_cast<uint8_t*>(codes), ldq, const_cast<float*>(scales), ceil_div(d, ckpt::kGroup)}, ldx, m, (int)d, (float)(1.0 / (double)d), mean, rstd, active,
                     weight, dx, alone ? dweight : (float*)workspace, alone ? dbias : (float*)workspace + d, 2 * d};
    const int item = dtype_size(dtype);
    int access = ckpt::access_of(dy, ldy, m, d, item), other = ckpt::access_of(dx, d, m, d, item);
    access = other < access ? other : access;
    if (x != nullptr) {
      other = ckpt::access_of(x, ldx, m, d, item);
      access = other < access ? other : access;
    }
    F2C_BY_ROWS(ln::run, dtype, access, a, how, st);
    if (const int rc = check_launch(op)) return rc;
  }
  if (alone) return F2C_OK;
  const int parts = m > 0 ? how.ctas : 0;
  launch_dependent(ln::join_kernel, dim3((unsigned)ceil_div(2 * d, 8)), 32 * (parts >= 512 ? 32 : parts / 16 + 1), 0, st, (const float*)workspace, parts, (int)d, dweight, dbias);
  return check_launch(op);
}
