// out [m, n] = act(s[i] ws[j] sum_t q[i, t] w[j, t] + b[j]) in 8-bit integers (f2c_int8_mm, f2c_int8_linear).
//
// One 64 x 64 tile of the output per CTA, 16 columns of both operands in shared memory at a time, four-element dot products.
#include "int8_mm.cuh"

namespace f2c {
namespace i8 {

constexpr int kTile = 64, kStep = 16, kThreads = 256;

struct Params {
  const int8_t *a, *b;
  int64_t lda, ldb;
  const float *a_scales, *b_scales, *bias;
  void* out;
  int64_t m, n, k;
  int relu;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) mm_kernel(const Params p) {
  dependency_wait();
  release_dependents();
  __shared__ __align__(16) int8_t as[kTile][kStep + 4], bs[kTile][kStep + 4];
  const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16;
  const int64_t row0 = (int64_t)blockIdx.x * kTile, col0 = (int64_t)blockIdx.y * kTile;
  int acc[4][4] = {};
  for (int64_t t0 = 0; t0 < p.k; t0 += kStep) {
    for (int e = tid; e < kTile * kStep; e += kThreads) {
      const int r = e / kStep, t = e % kStep;
      const bool in = t0 + t < p.k;
      as[r][t] = in && row0 + r < p.m ? p.a[(row0 + r) * p.lda + t0 + t] : 0;
      bs[r][t] = in && col0 + r < p.n ? p.b[(col0 + r) * p.ldb + t0 + t] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < kStep; q += 4)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __dp4a(*reinterpret_cast<const int*>(&as[ty + 16 * i][q]), *reinterpret_cast<const int*>(&bs[tx + 16 * j][q]), acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t r = row0 + ty + 16 * i, c = col0 + tx + 16 * j;
      if (r >= p.m || c >= p.n) continue;
      float v = (float)acc[i][j] * (p.a_scales[r] * p.b_scales[c]);
      if (p.bias != nullptr) v += p.bias[c];
      ((T*)p.out)[r * p.n + c] = from_float<T>(p.relu && v <= 0.0f ? 0.0f : v);
    }
}

static int check(const char* op, int64_t m, int64_t n, int64_t k, int out_dtype) {
  F2C_REQUIRE(m >= 0 && n >= 0 && k >= 0, F2C_ERR_INVALID, "%s: negative size", op);
  F2C_REQUIRE(is_float_dtype(out_dtype), F2C_ERR_UNSUPPORTED, "%s: the output must be float32, float16 or bfloat16", op);
  F2C_REQUIRE(k <= kMaxK, F2C_ERR_LIMIT, "%s: more than %d columns", op, kMaxK);
  F2C_REQUIRE(m <= kMaxRows && n <= (1 << 21), F2C_ERR_LIMIT, "%s: too many rows", op);
  return F2C_OK;
}

static int mm(const char* op, const Params& p, int out_dtype, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(p.m, kTile), (unsigned)ceil_div(p.n, kTile));
  auto* kern = out_dtype == F2C_F32 ? mm_kernel<float> : out_dtype == F2C_F16 ? mm_kernel<__half> : mm_kernel<__nv_bfloat16>;
  launch_dependent(kern, grid, kThreads, 0, st, p);
  return check_launch(op);
}

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

}  // namespace i8
}  // namespace f2c

using namespace f2c;

extern "C" int64_t f2c_int8_mm_workspace(const int8_t*, int64_t, const int8_t*, int64_t, int64_t, int64_t, int64_t) { return 0; }

extern "C" int f2c_int8_mm(const int8_t* codes, int64_t ldq, const float* scales, const int8_t* w, int64_t ldw, const float* w_scales,
                           const float* bias, int relu, void* out, int out_dtype, int64_t m, int64_t n, int64_t k, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  const char* op = "int8_mm";
  if (const int rc = i8::check(op, m, n, k, out_dtype)) return rc;
  F2C_REQUIRE((m <= 1 || ldq >= k) && (n <= 1 || ldw >= k), F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  if (m == 0 || n == 0) return F2C_OK;
  F2C_REQUIRE(out && scales && w_scales && (k == 0 || (codes && w)), F2C_ERR_INVALID, "%s: null pointer", op);
  return i8::mm(op, i8::Params{codes, w, ldq, ldw, scales, w_scales, bias, out, m, n, k, relu}, out_dtype, (cudaStream_t)stream);
}

extern "C" int64_t f2c_int8_linear_workspace(const int8_t*, int64_t, int64_t m, int64_t, int64_t k) {
  return m < 0 || k < 0 ? 0 : i8::round256(4 * m) + m * ((k + 15) / 16 * 16);
}

extern "C" int f2c_int8_linear(const void* x1, int64_t ld1, int64_t k1, const void* x2, int64_t ld2, int64_t k2, int dtype, const int8_t* w,
                               int64_t ldw, const float* w_scales, const float* bias, int relu, void* out, int out_dtype, int64_t m, int64_t n,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "int8_linear";
  const i8::Rows r{x1, x2, ld1, ld2, k1, k2, m, dtype};
  const int64_t k = k1 + k2;
  if (const int rc = i8::check_rows(op, r)) return rc;
  if (const int rc = i8::check(op, m, n, k, out_dtype)) return rc;
  F2C_REQUIRE(n <= 1 || ldw >= k, F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  if (m == 0 || n == 0) return F2C_OK;
  F2C_REQUIRE(out && w_scales && (k == 0 || w), F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(workspace && aligned(workspace, 256) && workspace_bytes >= f2c_int8_linear_workspace(w, ldw, m, n, k), F2C_ERR_INVALID,
              "%s: workspace too small or not 256-byte aligned", op);
  float* scales = (float*)workspace;
  int8_t* codes = (int8_t*)workspace + i8::round256(4 * m);
  const int64_t ldq = (k + 15) / 16 * 16;
  if (const int rc = i8::quantize(r, codes, ldq, scales, (cudaStream_t)stream)) return rc;
  return i8::mm(op, i8::Params{codes, w, ldq, ldw, scales, w_scales, bias, out, m, n, k, relu}, out_dtype, (cudaStream_t)stream);
}
