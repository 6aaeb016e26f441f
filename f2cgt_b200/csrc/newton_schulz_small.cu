// Newton-Schulz steps on matrices that one SM can hold: up to 128 x 256 (or transposed), each in a CTA, all of them in one launch (the weight matrices of a
// GraphSAGE network are of this size).
//
// X (its smaller side down, the larger one along) stays in shared memory as two planes of half precision, A and then R beside it; the sums are in
// TMEM: 128 columns for X X^T, 128 for A^2, 256 for R X.  X is laid out in pieces of 64 columns, rows of 128 bytes (128-byte swizzle): along K for
// X X^T, and the same bytes, read as rows along N, for R X.  A thread has a row of X, A and R and a quarter of its columns; what the next
// product reads goes from TMEM through registers to shared memory.
// What bounds it is the chain of 15 products, each with its MMAs, the reading of its sums and a barrier (128 x 128 float32: 24 MMAs of 64 cycles
// in some 2500).  Precision is as in newton_schulz.cu: float32 in pairs throughout, 16-bit matrices with A and R in one plane; X is always a pair.
#include "newton_schulz.cuh"

namespace f2c {
namespace nss {

using namespace ns;

constexpr int kThreads = 512, kRows = 128, kCols = 256;
constexpr int kPiece = kRows * 128;                                  // bytes of 64 columns of a plane
constexpr int kXPlane = kCols / 64 * kPiece, kAPlane = kRows / 64 * kPiece;
constexpr int kXAt = 0, kAAt = 2 * kXPlane, kBytes = kAAt + 2 * kAPlane;
constexpr int kPitch = kCols + 1;                                    // floats between rows of the result
static_assert(kRows * kPitch * 4 <= kBytes, "the result lies where X, A and R were");
constexpr uint32_t kGramAt = 0, kSquareAt = 128, kApplyAt = 256;     // columns of TMEM

struct Shared {
  uint64_t done;
  uint32_t tmem;
  int failed;
  double sums[kThreads / 32];
  Factors factors[F2C_MAX_NS_STEPS];
};

// Address of column c of row r of a plane at `plane`: eight columns are 16 bytes, the swizzle exchanges them with the row's.
__device__ __forceinline__ uint32_t place(uint32_t plane, int r, int c) {
  return plane + (uint32_t)((c >> 6) * kPiece + r * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4) + (c & 7) * 2);
}
__device__ __forceinline__ void store8(uint32_t at, const __half (&h)[8]) {
  union { __half h[8]; uint4 v; } u;
#pragma unroll
  for (int e = 0; e < 8; ++e) u.h[e] = h[e];
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(u.v.x), "r"(u.v.y), "r"(u.v.z), "r"(u.v.w) : "memory");
}
__device__ __forceinline__ void load8(uint32_t at, float (&v)[8]) {
  union { __half h[8]; uint32_t w[4]; } u;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.w[0]), "=r"(u.w[1]), "=r"(u.w[2]), "=r"(u.w[3]) : "r"(at) : "memory");
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __half2float(u.h[e]);
}
// eight columns from c on as half precision, and what that leaves
__device__ __forceinline__ void store_pair(uint32_t high, uint32_t low, bool both, int r, int c, const float (&v)[8]) {
  __half h[8], l[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    h[e] = __float2half_rn(v[e]);
    l[e] = __float2half_rn(v[e] - __half2float(h[e]));
  }
  store8(place(high, r, c), h);
  if (both) store8(place(low, r, c), l);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) small_kernel(const __grid_constant__ Matrices s, const __grid_constant__ Steps st, int64_t stack_rows, int64_t stack_cols, int* error) {
  constexpr bool kWide = sizeof(T) == 4;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Shared sh;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* const result = reinterpret_cast<float*>(smem_raw + (smem - smem_u32(smem_raw)));
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31, z = blockIdx.x;
  const int rows = (int)(s.listed ? s.list[z].rows : stack_rows), cols = (int)(s.listed ? s.list[z].cols : stack_cols), size = rows * cols;
  const bool tall = rows > cols;
  const int p = tall ? cols : rows, q = tall ? rows : cols, p16 = (p + 15) / 16 * 16, q16 = (q + 15) / 16 * 16;
  uint32_t left = kWaitLimit;

  if (wid == 0) alloc_tmem(&sh.tmem, 512);
  if (tid == 0) {
    init_bar(&sh.done, 1);
    fence_bars();
    sh.failed = 0;
  }
  for (int i = tid; i < kBytes / 16; i += kThreads)
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(smem + 16u * (uint32_t)i), "r"(0u) : "memory");
  dependency_wait();
  release_dependents();

  // ================= the norm, and X
  const T* const grad = s.template grad<T>(z);
  float* const momentum = s.moment(z);
  const bool nesterov = s.nesterov != 0;
  double sum = 0.0;
#pragma unroll 4
  for (int i = tid; i < size; i += kThreads) {
    float u = to_float(grad[i]);
    if (momentum != nullptr) {
      const float m = fmaf(s.mu, momentum[i], u);
      momentum[i] = m;
      u = nesterov ? fmaf(s.mu, m, u) : m;
    }
    sum = fma((double)u, (double)u, sum);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sh.sums[wid] = sum;
  fence_before();
  __syncthreads();
  fence_after();
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) sum += sh.sums[w];
  const double norm = sqrt(sum);
  const int up = scale_up(norm);
  if (tid == 0) make_factors(st, norm, up, sh.factors);
  const float by = power2(up / 2), more = norm <= 1e300 ? power2(up - up / 2) : __int_as_float(0x7fffffff);
#pragma unroll 4
  for (int i = tid; i < size; i += kThreads) {
    float u = to_float(grad[i]);
    if (momentum != nullptr) {
      const float m = momentum[i];
      u = nesterov ? fmaf(s.mu, m, u) : m;
    }
    const float v = u * by * more;
    const int row = i / cols, col = i - row * cols, r = tall ? col : row, c = tall ? row : col;
    const __half h = __float2half_rn(v), l = __float2half_rn(v - __half2float(h));
    const uint32_t at = place(smem + kXAt, r, c);
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(__half_as_ushort(h)) : "memory");
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + kXPlane), "h"(__half_as_ushort(l)) : "memory");
  }
  fence_async();
  __syncthreads();

  // ================= the steps
  const uint32_t tmem = sh.tmem;
  const bool issues = wid == 0 && elected() != 0u;
  const int quarter = wid & 3, group = wid >> 2, row = quarter * 32 + lane;  // a thread's row of X, A and R, and which columns of them
  const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
  uint32_t phase = 0;
  // A product of 128 rows and `n` columns over K, in 16s: planes by planes, the small ones first (see newton_schulz.cu).
  const auto product = [&](uint32_t acc, uint32_t a, int a_planes, uint32_t b, int b_planes, uint32_t b_plane, bool b_turned, int n, int k16) {
    if (wid == 0) {
      const bool go = issues && left != 0u;
      fence_after();
      const uint32_t idesc = instruction(kSumF32, kFormatF16, kRows, (uint32_t)n) | (b_turned ? kTurnedB : 0u);
      const uint32_t a_plane = a == smem + kXAt ? kXPlane : kAPlane;
      const uint32_t a_low = desc_low(a, kChunkAlongK), b_low = desc_low(b, b_turned ? kPiece : kChunkAlongK);
      bool on = false;
      for (int t = 0; t < a_planes + b_planes - 1; ++t) {
        const bool large = t + 2 == a_planes + b_planes, of_a = !large && t == 0 && a_planes > 1;
        const uint32_t at = a_low + (of_a ? a_plane >> 4 : 0u), bt = b_low + (large || of_a ? 0u : b_plane >> 4);
        for (int e = 0; e < k16; ++e, on = true) {  // 16 of K: 32 bytes of a row, 64 columns to a piece; turned: 16 rows
          const uint32_t along = (uint32_t)((e >> 2) * (kPiece >> 4) + (e & 3) * (int)kStepAlongK);
          mma_f16(go, acc, desc(at + along), desc(bt + (b_turned ? (uint32_t)e * kStepTurned : along)), idesc, on);
        }
      }
      commit(go, &sh.done);
    }
    wait_bar(&sh.done, phase & 1u, left);
    ++phase;
    __syncwarp();
    fence_after();
  };
  // what is written to shared memory is there for the next product, what was read from TMEM may be written over
  const auto next = [&]() {
    fence_async();
    fence_before();
    __syncthreads();
  };
  const int inner = kWide ? 2 : 1;
  float kept[kCols / 4];  // of the result: a thread's columns
#pragma unroll
  for (int j = 0; j < kCols / 4; ++j) kept[j] = 0.0f;
  for (int t = 0; t < st.count; ++t) {
    const Factors f = sh.factors[t];
    const bool poly = st.co[3 * t + 2] != 0.0f, last = t + 1 == st.count;
    // A = X X^T
    product(tmem + kGramAt, smem + kXAt, inner, smem + kXAt, inner, kXPlane, false, p16, q16 / 16);
    const int c0 = group * 32;  // of 128
    uint32_t a[32];
    if (c0 < p16) {
      tmem_ld32(lanes + kGramAt + (uint32_t)c0, a);
      tmem_wait(a);
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(a[j + e]) * f.gram;
        store_pair(smem + kAAt, smem + kAAt + kAPlane, kWide, row, c0 + j, v);
      }
    }
    next();
    if (poly) {  // R = c A^2 + b A
      product(tmem + kSquareAt, smem + kAAt, inner, smem + kAAt, inner, kAPlane, false, p16, p16 / 16);
      if (c0 < p16) {
        uint32_t r[32];
        tmem_ld32(lanes + kSquareAt + (uint32_t)c0, r);
        tmem_wait(r);
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = fmaf(f.poly_c, __uint_as_float(r[j + e]), f.poly_b * (__uint_as_float(a[j + e]) * f.gram));
          store_pair(smem + kAAt, smem + kAAt + kAPlane, kWide, row, c0 + j, v);
        }
      }
      next();
    }
    // X <- a X + R X: X's rows run along K here
    product(tmem + kApplyAt, smem + kAAt, inner, smem + kXAt, 2, kXPlane, true, q16, p16 / 16);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int x0 = group * 64 + half * 32;  // of 256
      if (x0 >= q16) continue;
      uint32_t r[32];
      tmem_ld32(lanes + kApplyAt + (uint32_t)x0, r);
      tmem_wait(r);
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        float h[8], l[8], v[8];
        load8(place(smem + kXAt, row, x0 + j), h);
        load8(place(smem + kXAt + kXPlane, row, x0 + j), l);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = fmaf(f.own, h[e], fmaf(f.own, l[e], __uint_as_float(r[j + e]) * f.apply));
          kept[half * 32 + j + e] = v[e];
        }
        if (!last) store_pair(smem + kXAt, smem + kXAt + kXPlane, true, row, x0 + j, v);
      }
    }
    if (!last) next();
  }
  if (st.count == 0) {
    const float kappa = sh.factors[0].apply;
#pragma unroll
    for (int j = 0; j < kCols / 4; j += 8) {
      float h[8], l[8];
      load8(place(smem + kXAt, row, group * 64 + j), h);
      load8(place(smem + kXAt + kXPlane, row, group * 64 + j), l);
#pragma unroll
      for (int e = 0; e < 8; ++e) kept[j + e] = kappa * (h[e] + l[e]);
    }
  }

  // ================= the result, as it lies in memory
  if (left == 0u) sh.failed = 1;
  fence_before();
  __syncthreads();
  const bool lost = sh.failed != 0;
#pragma unroll
  for (int j = 0; j < kCols / 4; ++j)
    if (row < p && group * 64 + j < q) result[row * kPitch + group * 64 + j] = kept[j];
  __syncthreads();
  T* const out = s.template result<T>(z);
  const float gain = s.listed ? s.gain(rows, cols) : 0.0f;
#pragma unroll 4
  for (int i = tid; i < size; i += kThreads) {
    const int r = i / cols, c = i - r * cols;
    float v = result[tall ? c * kPitch + r : r * kPitch + c];
    if (s.listed) v = s.keep * to_float(out[i]) - gain * v;
    out[i] = from_float<T>(lost ? __int_as_float(0x7fffffff) : v);
  }
  if (lost && wid == 0) {  // MMAs in flight read shared memory and write TMEM: wait (bounded) for them
    left = kWaitLimit;
    commit(issues, &sh.done);
    wait_bar(&sh.done, phase & 1u, left);
    __syncwarp();
  }
  if (wid == 0) {
    fence_after();
    free_tmem(tmem, 512);
  }
  if (lost && tid == 0) report_wait(error, 6);
}

template <typename T>
static int launch(const char* op, const Matrices& s, int count, int64_t rows, int64_t cols, const Steps& st, cudaStream_t stream) {
  auto* kern = small_kernel<T>;
  constexpr int bytes = kBytes + 1024;
  if (const int rc = allow_smem(op, (const void*)kern, bytes)) return rc;
  launch_dependent(kern, dim3((unsigned)count), kThreads, bytes, stream, s, st, rows, cols, stream_error_word());
  return check_launch(op);
}

}  // namespace nss

namespace ns {

bool is_small(int64_t rows, int64_t cols) {
  const int64_t p = rows < cols ? rows : cols, q = rows < cols ? cols : rows;
  return p <= nss::kRows && q <= nss::kCols;
}

int small(const char* op, const Matrices& s, int count, int64_t rows, int64_t cols, int dtype, const Steps& st, cudaStream_t stream) {
  if (dtype == F2C_F32) return nss::launch<float>(op, s, count, rows, cols, st, stream);
  if (dtype == F2C_F16) return nss::launch<__half>(op, s, count, rows, cols, st, stream);
  return nss::launch<__nv_bfloat16>(op, s, count, rows, cols, st, stream);
}

}  // namespace ns
}  // namespace f2c
