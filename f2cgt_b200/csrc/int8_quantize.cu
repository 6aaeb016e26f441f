// Codes and scales of rows (f2c_int8_quantize): scale = max|x| / 127, code = round-to-even(x / scale), both quotients as single
// precision has them, so that every implementation of the definition gives the same codes.
//
// Bound by reading the rows: a row's values stay in registers between its maximum and its codes.  A warp has a row, or a CTA where the
// row is too long for one warp's registers; loads are as wide as the rows' alignment allows.  The quotient is a product with the
// reciprocal, which is at most 127 * 3 * 2^-24 off; only where it lies so near to a tie that this could matter is the division made.
#include "int8_mm.cuh"

namespace f2c {
namespace i8q {

constexpr int kThreads = 256, kKept = 4;  // vectors of a row that a thread keeps

template <int BYTES> struct Raw;
template <> struct Raw<16> { using type = uint4; };
template <> struct Raw<4> { using type = uint32_t; };
template <> struct Raw<2> { using type = uint16_t; };
template <int BYTES> struct Out;
template <> struct Out<8> { using type = uint2; };
template <> struct Out<4> { using type = uint32_t; };
template <> struct Out<2> { using type = uint16_t; };
template <> struct Out<1> { using type = uint8_t; };

// BYTES of T's, V of them
template <typename T, int BYTES>
struct Vector {
  static constexpr int V = BYTES / (int)sizeof(T);
  using R = typename Raw<BYTES>::type;
  union { R raw; T v[V]; };
  __device__ __forceinline__ Vector() : raw() {}
};

// The code of v, in the low byte.  inv 0: divide.
__device__ __forceinline__ uint32_t code_of(float v, float scale, float inv) {
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to even and leaves the integer in the low bits
  const float t = v * inv, shifted = t + kRound;
  uint32_t code = __float_as_uint(shifted);
  if (inv == 0.0f || fabsf(t - (shifted - kRound)) > 0.4999f)
    code = __float_as_uint(fminf(fmaxf(rintf(__fdiv_rn(v, scale)), -127.0f), 127.0f) + kRound);
  return code & 0xffu;
}

template <typename T, int BYTES, int THREADS>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const i8::Rows r, int8_t* __restrict__ codes, int64_t ldq, float* __restrict__ scales) {
  using Vec = Vector<T, BYTES>;
  constexpr int V = Vec::V;
  using O = typename Out<V>::type;
  dependency_wait();
  release_dependents();
  const int at = threadIdx.x % THREADS;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / THREADS) + threadIdx.x / THREADS;
  if (row >= r.m) return;  // all threads of a warp
  const int n1 = (int)(r.k1 / V), n = n1 + (int)(r.k2 / V);
  const typename Vec::R* x1 = reinterpret_cast<const typename Vec::R*>((const T*)r.x1 + row * r.ld1);
  const typename Vec::R* x2 = reinterpret_cast<const typename Vec::R*>((const T*)r.x2 + row * r.ld2) - n1;
  auto read = [&](int i) {
    Vec v;
    v.raw = __ldg(i < n1 ? x1 + i : x2 + i);
    return v;
  };
  float top = 0.0f;
  bool bad = false;
  auto look = [&](const Vec& v) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = fabsf(to_float(v.v[e]));
      bad |= !(a <= 3.4028235e38f);
      top = fmaxf(top, a);
    }
  };
  Vec kept[kKept];
#pragma unroll
  for (int q = 0; q < kKept; ++q)
    if (at + q * THREADS < n) kept[q] = read(at + q * THREADS);
#pragma unroll
  for (int q = 0; q < kKept; ++q) look(kept[q]);
  for (int i = at + kKept * THREADS; i < n; i += THREADS) look(read(i));
  uint32_t bits = bad ? 0xffffffffu : __float_as_uint(top);
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (THREADS > 32) {
    __shared__ uint32_t of_warp[kThreads / 32];
    if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) bits = max(bits, of_warp[w]);
  }
  bad = bits == 0xffffffffu;
  const float scale = bad ? __int_as_float(0x7fffffff) : __fdiv_rn(__uint_as_float(bits), 127.0f);
  const bool zero = bad || scale == 0.0f;
  const float inv = zero || scale < 1e-37f ? 0.0f : __frcp_rn(scale);  // (the reciprocal of less has no place, or few bits)
  O* out = reinterpret_cast<O*>(codes + row * ldq);
  auto write = [&](int i, const Vec& v) {
    uint32_t word[V > 4 ? 2 : 1] = {};
    if (!zero) {
#pragma unroll
      for (int e = 0; e < V; ++e) word[e / 4] |= code_of(to_float(v.v[e]), scale, inv) << (e % 4 * 8);
    }
    if constexpr (V == 8) out[i] = make_uint2(word[0], word[1]);
    else out[i] = (O)word[0];
  };
#pragma unroll
  for (int q = 0; q < kKept; ++q)
    if (at + q * THREADS < n) write(at + q * THREADS, kept[q]);
  for (int i = at + kKept * THREADS; i < n; i += THREADS) write(i, read(i));
  if (at == 0) scales[row] = scale;
}

template <typename T, int BYTES>
static void launch(const i8::Rows& r, int8_t* codes, int64_t ldq, float* scales, cudaStream_t st) {
  if ((r.k1 + r.k2) * (int64_t)sizeof(T) > 32 * kKept * BYTES)
    launch_dependent(quantize_kernel<T, BYTES, kThreads>, dim3((unsigned)r.m), kThreads, 0, st, r, codes, ldq, scales);
  else
    launch_dependent(quantize_kernel<T, BYTES, 32>, dim3((unsigned)ceil_div(r.m, kThreads / 32)), kThreads, 0, st, r, codes, ldq, scales);
}

// Rows whose starts and lengths, and those of their codes, allow reads of `bytes`.
template <typename T>
static bool fits(const i8::Rows& r, const int8_t* codes, int64_t ldq, int bytes) {
  const int64_t v = bytes / (int64_t)sizeof(T);
  return aligned(r.x1, bytes) && aligned(r.x2, bytes) && aligned(codes, v) && r.k1 % v == 0 && r.k2 % v == 0 &&
         (r.m <= 1 || (r.ld1 % v == 0 && r.ld2 % v == 0 && ldq % v == 0));
}

template <typename T>
static void any(const i8::Rows& r, int8_t* codes, int64_t ldq, float* scales, cudaStream_t st) {
  if (fits<T>(r, codes, ldq, 16)) return launch<T, 16>(r, codes, ldq, scales, st);
  if constexpr (sizeof(T) == 2) {
    if (!fits<T>(r, codes, ldq, 4)) return launch<T, 2>(r, codes, ldq, scales, st);
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
