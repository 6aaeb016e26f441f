// Newton-Schulz steps on matrices that one SM can hold: up to 128 x 256 (or transposed), each in a CTA, all of them in one launch (the weight matrices of a
// GraphSAGE network of 128 columns are of this size; those of 256 x 256 are not).
//
// X (its smaller side down, the larger one along) stays in shared memory as two planes of half precision, A and then R beside it; the sums are in
// TMEM: 128 columns for X X^T, 128 for A^2, 256 for R X.  X is laid out in pieces of 64 columns, rows of 128 bytes (128-byte swizzle): along K for
// X X^T, and the same bytes, read as rows along N, for R X.  A thread has a row of X, A and R and a quarter of its columns; what the next
// product reads goes from TMEM through registers to shared memory.
// What bounds it is the chain of 15 products, each with its MMAs, the reading of its sums and a barrier (128 x 128 float32: five steps 43.5 us, so 2.8 us
// or some 5300 cycles a product, of which its 24 MMAs take 64 each).  Precision is as in newton_schulz.cu: everything in pairs, but that bfloat16's
// X X^T takes the high planes alone.
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
  uint64_t done, drain;
  uint32_t tmem;
  int failed;
  double sums[kThreads / 32];
  Factors factors[F2C_MAX_NS_STEPS];
};

// Address of column c of row r of a plane at `plane`: eight columns are 16 bytes, the swizzle exchanges them with the row's.
__device__ __forceinline__ uint32_t place(uint32_t plane, int r, int c) {
  return plane + (uint32_t)((c >> 6) * kPiece + r * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4) + (c & 7) * 2);
}
// Eight columns from c on as half precision, and what that leaves.
__device__ __forceinline__ void split2(float x, float y, uint32_t& high, uint32_t& low) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  high = *reinterpret_cast<const uint32_t*>(&h);
  low = *reinterpret_cast<const uint32_t*>(&l);
}
__device__ __forceinline__ void store_pair(uint32_t high, uint32_t low, int r, int c, const float (&v)[8]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) split2(v[2 * e], v[2 * e + 1], h[e], l[e]);
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(place(high, r, c)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(place(low, r, c)), "r"(l[0]), "r"(l[1]), "r"(l[2]), "r"(l[3]) : "memory");
}
__device__ __forceinline__ void load8(uint32_t at, float (&v)[8]) {
  uint32_t w[4];
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
    v[2 * e] = f.x;
    v[2 * e + 1] = f.y;
  }
}

// V elements of a matrix, which lie in one row of it
template <typename T, int V> struct alignas(V * sizeof(T)) Few { T v[V]; };

// V: elements read and written at a time
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 1) small_kernel(const __grid_constant__ Matrices s, const __grid_constant__ Steps st, int64_t stack_rows, int64_t stack_cols, int* error) {
  constexpr bool kWide = is_wide<T>;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Shared sh;
  const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
  float* const result = reinterpret_cast<float*>(smem_raw + (smem - smem_u32(smem_raw)));
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31, z = blockIdx.x;
  const int rows = (int)(s.listed ? s.list[z].rows : stack_rows), cols = (int)(s.listed ? s.list[z].cols : stack_cols), size = rows * cols;
  const bool tall = rows > cols;
  const int p = tall ? cols : rows, q = tall ? rows : cols, p16 = (p + 15) / 16 * 16, q16 = (q + 15) / 16 * 16;
  uint32_t left = st.tries;

  if (wid == 0) alloc_tmem(&sh.tmem, 512);
  if (tid == 0) {
    init_bar(&sh.done, 1);
    init_bar(&sh.drain, 1);
    fence_bars();
    sh.failed = 0;
  }
  for (int i = tid; i < kBytes / 16; i += kThreads)
    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(smem + 16u * (uint32_t)i), "r"(0u) : "memory");
  dependency_wait();
  if (wid == 0) release_dependents();  // the warp that has allocated

  // ================= the norm, and X: a thread's elements stay in registers in between
  const T* const grad = s.template grad<T>(z);
  float* const momentum = s.moment(z);
  constexpr int kMost = kRows * kCols / kThreads / V, kBlock = kMost < 16 ? kMost / 2 : 16;  // of a thread, and on their way at once
  const int count = size / V;
  float u[kMost][V];
  double sum = 0.0;
#pragma unroll
  for (int b = 0; b < kMost; b += kBlock) {
    if (b * kThreads >= count) break;
#pragma unroll
    for (int j = b; j < b + kBlock; ++j) {
      Few<T, V> g{};
      if (j * kThreads + tid < count) g = reinterpret_cast<const Few<T, V>*>(grad)[j * kThreads + tid];
#pragma unroll
      for (int e = 0; e < V; ++e) u[j][e] = to_float(g.v[e]);
    }
    if (momentum != nullptr) {
      Few<float, V> m[kBlock];
#pragma unroll
      for (int j = 0; j < kBlock; ++j)
        if ((b + j) * kThreads + tid < count) m[j] = reinterpret_cast<const Few<float, V>*>(momentum)[(b + j) * kThreads + tid];
#pragma unroll
      for (int j = 0; j < kBlock; ++j) {
        if ((b + j) * kThreads + tid >= count) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          m[j].v[e] = fmaf(s.mu, m[j].v[e], u[b + j][e]);
          u[b + j][e] = s.nesterov ? fmaf(s.mu, m[j].v[e], u[b + j][e]) : m[j].v[e];
        }
        reinterpret_cast<Few<float, V>*>(momentum)[(b + j) * kThreads + tid] = m[j];
      }
    }
#pragma unroll
    for (int j = b; j < b + kBlock; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) sum = fma((double)u[j][e], (double)u[j][e], sum);
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
  // V elements from i on are at (i / cols, i % cols); from one of a thread's to the next the pair moves by a fixed one
  const int first_r = tid * V / cols, first_c = tid * V - first_r * cols, dr = kThreads * V / cols, dc = kThreads * V - dr * cols;
  int r = first_r, c = first_c;
  const auto move = [&]() {
    r += dr;
    c += dc;
    if (c >= cols) {
      c -= cols;
      ++r;
    }
  };
#pragma unroll
  for (int b = 0; b < kMost; b += kBlock) {
    if (b * kThreads >= count) break;
#pragma unroll
    for (int j = b; j < b + kBlock; ++j, move()) {
      if (j * kThreads + tid >= count) continue;
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = u[j][e] * by * more;
      if constexpr (V == 4) {
        uint32_t h[2], l[2];
        split2(v[0], v[1], h[0], l[0]);
        split2(v[2], v[3], h[1], l[1]);
        if (!tall) {
          const uint32_t at = place(smem + kXAt, r, c);
          asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(h[0]), "r"(h[1]) : "memory");
          asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at + kXPlane), "r"(l[0]), "r"(l[1]) : "memory");
        } else {  // four rows: every lane starts with another of them, so that 32 lanes meet eight bank groups
          const int turn = (lane >> 1) & 3;
          const uint64_t h4 = (uint64_t)h[1] << 32 | h[0], l4 = (uint64_t)l[1] << 32 | l[0];
          const uint64_t hr = turn == 0 ? h4 : h4 >> (16 * turn) | h4 << (64 - 16 * turn), lr = turn == 0 ? l4 : l4 >> (16 * turn) | l4 << (64 - 16 * turn);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t at = place(smem + kXAt, c + ((e + turn) & 3), r);
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"((uint16_t)(hr >> (16 * e))) : "memory");
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + kXPlane), "h"((uint16_t)(lr >> (16 * e))) : "memory");
          }
        }
      } else {
        uint32_t h, l;
        split2(v[0], 0.0f, h, l);
        const uint32_t at = place(smem + kXAt, tall ? c : r, tall ? r : c);
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"((uint16_t)h) : "memory");
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + kXPlane), "h"((uint16_t)l) : "memory");
      }
    }
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
      const uint32_t b_step = b_turned ? kStepTurned : kStepAlongK;
      bool on = false;
      for (int t = 0; t < a_planes + b_planes - 1; ++t) {
        const bool large = t + 2 == a_planes + b_planes, of_a = !large && t == 0 && a_planes > 1;
        const uint32_t at = a_low + (of_a ? a_plane >> 4 : 0u), bt = b_low + (large || of_a ? 0u : b_plane >> 4);
        uint32_t ae = at, be = bt;
        int e = 0;
        for (; e + 4 <= k16; e += 4, ae += kPiece >> 4, be += b_turned ? 4 * kStepTurned : kPiece >> 4, on = true) {  // a piece, or 64 rows of one
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)  // 16 of K: 32 bytes of a row; turned: 16 rows
            mma_f16(go, acc, desc(ae + i * kStepAlongK), desc(be + i * b_step), idesc, on || i != 0);
        }
        for (; e < k16; ++e, ae += kStepAlongK, be += b_step, on = true) mma_f16(go, acc, desc(ae), desc(be), idesc, on);
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
  constexpr int kGramPlanes = kWide ? 2 : 1;
  float kept[kCols / 4];  // of the result: a thread's columns
#pragma unroll
  for (int j = 0; j < kCols / 4; ++j) kept[j] = 0.0f;
  for (int t = 0; t < st.count; ++t) {
    const Factors f = sh.factors[t];
    const bool poly = st.co[3 * t + 2] != 0.0f, last = t + 1 == st.count;
    // A = X X^T
    product(tmem + kGramAt, smem + kXAt, kGramPlanes, smem + kXAt, kGramPlanes, kXPlane, false, p16, q16 / 16);
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
        store_pair(smem + kAAt, smem + kAAt + kAPlane, row, c0 + j, v);
      }
    }
    next();
    if (poly) {  // R = c A^2 + b A
      product(tmem + kSquareAt, smem + kAAt, 2, smem + kAAt, 2, kAPlane, false, p16, p16 / 16);
      if (c0 < p16) {
        uint32_t r[32];
        tmem_ld32(lanes + kSquareAt + (uint32_t)c0, r);
        tmem_wait(r);
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = fmaf(f.poly_c, __uint_as_float(r[j + e]), f.poly_b * (__uint_as_float(a[j + e]) * f.gram));
          store_pair(smem + kAAt, smem + kAAt + kAPlane, row, c0 + j, v);
        }
      }
      next();
    }
    // X <- a X + R X: X's rows run along K here
    product(tmem + kApplyAt, smem + kAAt, 2, smem + kXAt, 2, kXPlane, true, q16, p16 / 16);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int x0 = (group + 4 * half) * 32;  // of 256
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
        if (!last) store_pair(smem + kXAt, smem + kXAt + kXPlane, row, x0 + j, v);
      }
    }
    if (!last) next();
  }
  if (st.count == 0) {
    const float kappa = sh.factors[0].apply;
#pragma unroll
    for (int j = 0; j < kCols / 4; j += 8) {
      float h[8], l[8];
      load8(place(smem + kXAt, row, (group + 4 * (j >> 5)) * 32 + (j & 31)), h);
      load8(place(smem + kXAt + kXPlane, row, (group + 4 * (j >> 5)) * 32 + (j & 31)), l);
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
  for (int j = 0; j < kCols / 4; ++j) {
    const int column = (group + 4 * (j >> 5)) * 32 + (j & 31);
    if (row < p && column < q) result[row * kPitch + column] = kept[j];
  }
  __syncthreads();
  T* const out = s.template result<T>(z);
  const float gain = s.listed ? s.gain(rows, cols) : 0.0f, nan = __int_as_float(0x7fffffff);
  r = first_r;
  c = first_c;
#pragma unroll
  for (int b = 0; b < kMost; b += kBlock) {
    if (b * kThreads >= count) break;
    Few<T, V> w[kBlock];
    if (s.listed) {
#pragma unroll
      for (int j = 0; j < kBlock; ++j)
        if ((b + j) * kThreads + tid < count) w[j] = reinterpret_cast<const Few<T, V>*>(out)[(b + j) * kThreads + tid];
    }
#pragma unroll
    for (int j = 0; j < kBlock; ++j, move()) {
      if ((b + j) * kThreads + tid >= count) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float v = result[tall ? (c + e) * kPitch + r : r * kPitch + c + e];
        if (s.listed) v = s.keep * to_float(w[j].v[e]) - gain * v;
        w[j].v[e] = from_float<T>(lost ? nan : v);
      }
      reinterpret_cast<Few<T, V>*>(out)[(b + j) * kThreads + tid] = w[j];
    }
  }
  if (lost && st.tries != 0u && wid == 0) {  // MMAs in flight read shared memory and write TMEM: wait (bounded) for them
    left = st.tries;
    commit(issues, &sh.drain);
    wait_bar(&sh.drain, 0, left);
    __syncwarp();
  }
  if (wid == 0) {
    fence_after();
    free_tmem(tmem, 512);
  }
  if (lost && tid == 0) report_wait(error, 6);
}

template <typename T, int V>
static int launch(const char* op, const Matrices& s, int count, int64_t rows, int64_t cols, const Steps& st, cudaStream_t stream) {
  auto* kern = small_kernel<T, V>;
  constexpr int bytes = kBytes + 1024;
  if (const int rc = allow_smem(op, (const void*)kern, bytes)) return rc;
  launch_dependent(kern, dim3((unsigned)count), kThreads, bytes, stream, s, st, rows, cols, stream_error_word());
  return check_launch(op);
}

template <typename T>
static int by_width(const char* op, const Matrices& s, int count, int64_t rows, int64_t cols, const Steps& st, cudaStream_t stream) {
  bool four = s.listed || (cols % 4 == 0 && aligned(s.g, 4 * sizeof(T)) && aligned(s.out, 4 * sizeof(T)));
  for (int i = 0; i < s.listed; ++i) {
    const f2c_muon_matrix& m = s.list[i];
    four = four && m.cols % 4 == 0 && aligned(m.grad, 4 * sizeof(T)) && aligned(m.weight, 4 * sizeof(T)) && aligned(m.momentum, 16);
  }
  return four ? launch<T, 4>(op, s, count, rows, cols, st, stream) : launch<T, 1>(op, s, count, rows, cols, st, stream);
}

}  // namespace nss

namespace ns {

bool is_small(int64_t rows, int64_t cols) {
  const int64_t p = rows < cols ? rows : cols, q = rows < cols ? cols : rows;
  return p <= nss::kRows && q <= nss::kCols;
}

int small(const char* op, const Matrices& s, int count, int64_t rows, int64_t cols, int dtype, const Steps& st, cudaStream_t stream) {
  if (dtype == F2C_F32) return nss::by_width<float>(op, s, count, rows, cols, st, stream);
  if (dtype == F2C_F16) return nss::by_width<__half>(op, s, count, rows, cols, st, stream);
  return nss::by_width<__nv_bfloat16>(op, s, count, rows, cols, st, stream);
}

}  // namespace ns
}  // namespace f2c
