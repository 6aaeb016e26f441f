// Codes and scales of rows (f2c_int8_quantize): scale = max|x| / 127, code = round-to-even(x / scale), both quotients as single
// precision has them, so that every implementation of the definition gives the same codes.
//
// Bound by reading the rows (59,000 x 256 float32: 14.5 us, 5.2 TB/s): a row's values stay in registers between its maximum and its codes.  A warp has a row, or a CTA where the
// row is too long for one warp's registers; loads are as wide as the rows' alignment allows.  The quotient is a product with the
// reciprocal, which is at most 127 * 3 * 2^-24 off; only where it lies so near to a tie that this could matter is the division made.
#include "int8_mm.cuh"

namespace f2c {
namespace i8q {

constexpr int kThreads = 256;

// THREADS per row, of whose vectors each keeps KEPT
template <typename T, int BYTES, int THREADS, int KEPT>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const i8::Rows r, int8_t* __restrict__ codes, int64_t ldq, float* __restrict__ scales) {
  using Vec = i8::Vector<T, BYTES>;
  using R = typename i8::Words<BYTES>::type;
  constexpr int V = Vec::V;
  dependency_wait();
  release_dependents();
  const int at = threadIdx.x % THREADS;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / THREADS) + threadIdx.x / THREADS;
  if (row >= r.m) return;  // all threads of a warp
  const int n1 = (int)(r.k1 / V), n = n1 + (int)(r.k2 / V);
  const R* x1 = reinterpret_cast<const R*>((const T*)r.x1 + row * r.ld1);
  const R* x2 = reinterpret_cast<const R*>((const T*)r.x2 + row * r.ld2) - n1;
  auto read = [&](int i) {
    Vec v;
    v.raw = __ldg(i < n1 ? x1 + i : x2 + i);
    return v;
  };
  i8::Largest<T> part;
  auto look = [&](const Vec& v) {
#pragma unroll
    for (int e = 0; e < Vec::W; ++e) part.add(v.w[e]);
  };
  Vec kept[KEPT];
#pragma unroll
  for (int q = 0; q < KEPT; ++q)
    if (at + q * THREADS < n) kept[q] = read(at + q * THREADS);
#pragma unroll
  for (int q = 0; q < KEPT; ++q) look(kept[q]);
  for (int i = at + KEPT * THREADS; i < n; i += THREADS) look(read(i));
  uint32_t largest = __reduce_max_sync(0xffffffffu, part.of_float());
  if (THREADS > 32) {
    __shared__ uint32_t of_warp[kThreads / 32];
    if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) largest = max(largest, of_warp[w]);
  }
  const i8::Scale s = i8::scale_of(largest);
  int8_t* out = codes + row * ldq;
  // of vectors at, at + THREADS, ...: G at a time
  const auto left = [&](int i) { return i < n ? (n - i + THREADS - 1) / THREADS : 0; };
#pragma unroll
  for (int q = 0; q < KEPT; q += Vec::G)
    if (at + q * THREADS < n) i8::write<T, BYTES>(out + (at + q * THREADS) * V, THREADS * V, left(at + q * THREADS), kept + q, s);
  for (int i = at + KEPT * THREADS; i < n; i += Vec::G * THREADS) {
    Vec v[Vec::G];
#pragma unroll
    for (int g = 0; g < Vec::G; ++g)
      if (i + g * THREADS < n) v[g] = read(i + g * THREADS);
    i8::write<T, BYTES>(out + i * V, THREADS * V, left(i), v, s);
  }
  if (at == 0) scales[row] = s.scale;
}

// two vectors a lane, or as many as are encoded together
template <typename T, int BYTES> struct Vec2 { static constexpr int kept = i8::Vector<T, BYTES>::G > 2 ? 4 : 2; };

template <typename T, int BYTES>
static void launch(const i8::Rows& r, int8_t* codes, int64_t ldq, float* scales, cudaStream_t st) {
  const int64_t vectors = (r.k1 + r.k2) * (int64_t)sizeof(T) / BYTES;
  const dim3 warps((unsigned)ceil_div(r.m, kThreads / 32));
  // A row up to 16 vectors a lane long is a warp's; where rows are few, one of more than four vectors a lane has a CTA.
  if (vectors > 512 || (vectors > 128 && r.m < 1024))
    launch_dependent(quantize_kernel<T, BYTES, kThreads, 4>, dim3((unsigned)r.m), kThreads, 0, st, r, codes, ldq, scales);
  else if (vectors <= 64)
    launch_dependent(quantize_kernel<T, BYTES, 32, Vec2<T, BYTES>::kept>, warps, kThreads, 0, st, r, codes, ldq, scales);
  else if (vectors <= 128)
    launch_dependent(quantize_kernel<T, BYTES, 32, 4>, warps, kThreads, 0, st, r, codes, ldq, scales);
  else
    launch_dependent(quantize_kernel<T, BYTES, 32, 16>, warps, kThreads, 0, st, r, codes, ldq, scales);
}

template <typename T>
static void any(const i8::Rows& r, int8_t* codes, int64_t ldq, float* scales, cudaStream_t st) {
  if (r.fits(16, codes, ldq)) return launch<T, 16>(r, codes, ldq, scales, st);
  if (r.fits(8, codes, ldq)) return launch<T, 8>(r, codes, ldq, scales, st);
  if constexpr (sizeof(T) == 2) {
    if (!r.fits(4, codes, ldq)) return launch<T, 2>(r, codes, ldq, scales, st);
  }
  launch<T, 4>(r, codes, ldq, scales, st);
}

}  // namespace i8q

namespace i8 {

int quantize(const Rows& r, int8_t* codes, int64_t ldq, float* scales, cudaStream_t st) {
  if (r.dtype == F2C_F32) i8q::any<float>(r, codes, ldq, scales, st);
  else if (r.dtype == F2C_F16) i8q::any<__half>(r, codes, ldq, scales, st);
  else i8q::any<__nv_bfloat16>(r, codes, ldq, scales, st);
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
