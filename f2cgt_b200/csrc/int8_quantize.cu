// Codes and scales of rows (f2c_int8_quantize): scale = max|x| / 127, code = round-to-even(x / scale), both quotients as single
// precision has them, so that every implementation of the definition gives the same codes.
//
// A warp reads a row twice (the second time from L1 / L2).
#include "int8_mm.cuh"

namespace f2c {
namespace i8q {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const i8::Rows r, int8_t* __restrict__ codes, int64_t ldq, float* __restrict__ scales) {
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= r.m) return;
  const T* x1 = (const T*)r.x1 + row * r.ld1;
  const T* x2 = (const T*)r.x2 + row * r.ld2 - r.k1;
  const int64_t k = r.k1 + r.k2;
  float top = 0.0f;
  bool bad = false;
  for (int64_t t = lane; t < k; t += 32) {
    const float v = fabsf(to_float(t < r.k1 ? x1[t] : x2[t]));
    bad |= !(v <= 3.4028235e38f);
    top = fmaxf(top, v);
  }
  bad = __any_sync(0xffffffffu, bad);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float scale = bad ? __int_as_float(0x7fffffff) : __fdiv_rn(top, 127.0f);
  const bool zero = bad || scale == 0.0f;
  for (int64_t t = lane; t < k; t += 32) {
    const float v = to_float(t < r.k1 ? x1[t] : x2[t]);
    codes[row * ldq + t] = zero ? 0 : (int8_t)fminf(fmaxf(rintf(__fdiv_rn(v, scale)), -127.0f), 127.0f);
  }
  if (lane == 0) scales[row] = scale;
}

}  // namespace i8q

namespace i8 {

int quantize(const Rows& r, int8_t* codes, int64_t ldq, float* scales, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(r.m, i8q::kThreads / 32));
  auto* kern = r.dtype == F2C_F32 ? i8q::quantize_kernel<float> : r.dtype == F2C_F16 ? i8q::quantize_kernel<__half> : i8q::quantize_kernel<__nv_bfloat16>;
  launch_dependent(kern, grid, i8q::kThreads, 0, st, r, codes, ldq, scales);
  return check_launch("int8_quantize");
}

int check_rows(const char* op, const Rows& r) {
  F2C_REQUIRE(is_float_dtype(r.dtype), F2C_ERR_UNSUPPORTED, "%s: rows must be float32, float16 or bfloat16", op);
  F2C_REQUIRE(r.m >= 0 && r.k1 >= 0 && r.k2 >= 0, F2C_ERR_INVALID, "%s: negative size", op);
  F2C_REQUIRE(r.k1 + r.k2 <= kMaxK, F2C_ERR_LIMIT, "%s: more than %d columns", op, kMaxK);
  F2C_REQUIRE(r.m <= kMaxRows, F2C_ERR_LIMIT, "%s: too many rows", op);
  F2C_REQUIRE(r.m <= 1 || (r.ld1 >= r.k1 && r.ld2 >= r.k2), F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  F2C_REQUIRE(r.m == 0 || ((r.k1 == 0 || r.x1) && (r.k2 == 0 || r.x2)), F2C_ERR_INVALID, "%s: null pointer", op);
  return F2C_OK;
}

}  // namespace i8
}  // namespace f2c

using namespace f2c;

extern "C" int f2c_int8_quantize(const void* x1, int64_t ld1, int64_t k1, const void* x2, int64_t ld2, int64_t k2, int dtype, int64_t m,
                                 int8_t* codes, int64_t ldq, float* scales, void* stream) {
  const char* op = "int8_quantize";
  const i8::Rows r{x1, x2, ld1, ld2, k1, k2, m, dtype};
  if (const int rc = i8::check_rows(op, r)) return rc;
  if (m == 0) return F2C_OK;
  F2C_REQUIRE(scales && (codes || k1 + k2 == 0), F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(m == 1 || ldq >= k1 + k2, F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  return i8::quantize(r, codes, ldq, scales, (cudaStream_t)stream);
}
