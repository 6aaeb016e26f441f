// Activations to 8 bits and back (f2c_checkpoint_int8, f2c_checkpoint_values).  Back: bound by memory (8192 x 4096 bfloat16 19 us, 5.3 TB/s).  To 8 bits: by
// instructions, some hundred a group of a warp for 4 values a lane (the same 34 us, 2.9 TB/s; 59,000 x 128 float32 10.9 us, 3.5 TB/s).
//
// A warp has a group - 128 columns of a row - four columns a lane: its extremes are one reduction instruction each, its codes 128 bytes
// side by side, and every lane works out the step and its reciprocal.  Groups are taken kAhead at a time, all loads before the first use; lane a writes group a's step.
#include "checkpoint.cuh"

namespace f2c {
namespace ckpt {

constexpr int kThreads = 256, kWarps = kThreads / 32, kAhead = 4;

struct Place { int64_t row; int group; };
// group number `i` of all rows' groups (2^31 at most), and the one behind it
__device__ __forceinline__ Place place_of(int64_t i, uint32_t groups) { return Place{(int64_t)((uint32_t)i / groups), (int)((uint32_t)i % groups)}; }
__device__ __forceinline__ Place behind(Place p, int groups) { return p.group + 1 < groups ? Place{p.row, p.group + 1} : Place{p.row + 1, 0}; }

// EVEN: all groups have 128 columns
template <typename T, int ACCESS, bool EVEN>
__global__ void __launch_bounds__(kThreads) encode_kernel(const T* __restrict__ x, int64_t ldx, int64_t m, int d, Codes out) {
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t total = m * out.groups, first = ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * kAhead;
  Four<T, ACCESS> v[kAhead];
  Place at[kAhead];
  at[0] = place_of(first, (uint32_t)out.groups);
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    if (a > 0) at[a] = behind(at[a - 1], (int)out.groups);
    const int col = at[a].group * kGroup + 4 * lane;
    v[a].load(x + at[a].row * ldx + col, first + a < total ? (EVEN ? 4 : d - col) : 0);
  }
  Scale mine{0.0f, 0.0f};  // lane a: of group a
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    if (first + a >= total) break;
    f32x2 f[2];
    v[a].get(f);
    Scale s;
    const int col = at[a].group * kGroup + 4 * lane;
    const uint32_t codes = encode(f, EVEN ? 4 : d - col, s);
    // rows have room for whole 16 bytes: a word that starts in front of the row's end is there
    if (EVEN || col < d) *reinterpret_cast<uint32_t*>(out.codes + at[a].row * out.ld + col) = codes;
    if (lane == a) mine = s;
  }
  if (lane < kAhead && first + lane < total) store_scale(out.scales + 2 * (first + lane), mine);
}

template <typename T, int ACCESS>
__global__ void __launch_bounds__(kThreads) values_kernel(const Codes in, T* __restrict__ out, int64_t ldo, int64_t m, int d) {
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t total = m * in.groups, first = ((int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5)) * kAhead;
  uint32_t codes[kAhead];
  Scale s[kAhead];
  Place at[kAhead];
  at[0] = place_of(first, (uint32_t)in.groups);
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    if (a > 0) at[a] = behind(at[a - 1], (int)in.groups);
    const int col = at[a].group * kGroup + 4 * lane;
    if (first + a < total) {
      codes[a] = ldg_nc_u32_if(in.codes + at[a].row * in.ld + col, col < d);
      s[a] = load_scale(in.scales + 2 * (first + a));
    }
  }
#pragma unroll
  for (int a = 0; a < kAhead; ++a) {
    if (first + a >= total) return;
    f32x2 f[2];
    decode(codes[a], s[a], f);
    Four<T, ACCESS> v;
    v.set(f);
    const int col = at[a].group * kGroup + 4 * lane;
    v.store(out + at[a].row * ldo + col, d - col);
  }
}

int check_sizes(const char* op, int dtype, int64_t m, int64_t d) {
  F2C_REQUIRE(is_float_dtype(dtype), F2C_ERR_UNSUPPORTED, "%s: rows must be float32, float16 or bfloat16", op);
  F2C_REQUIRE(m >= 0 && d >= 0, F2C_ERR_INVALID, "%s: negative size", op);
  F2C_REQUIRE(m <= kMaxRows && d <= kMaxColumns, F2C_ERR_LIMIT, "%s: more than 2^31 rows or 2^20 columns", op);
  return F2C_OK;
}

int check_codes(const char* op, const uint8_t* codes, int64_t ldq, const float* scales, int64_t m, int64_t d) {
  if (m == 0 || d == 0) return F2C_OK;
  F2C_REQUIRE(codes && scales, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(aligned(codes, 16) && ldq % 16 == 0 && ldq >= d, F2C_ERR_INVALID, "%s: rows of codes must start on 16 bytes, with room for whole 16 bytes", op);
  F2C_REQUIRE(aligned(scales, 8), F2C_ERR_INVALID, "%s: scales must start on 8 bytes", op);
  return F2C_OK;
}

template <typename T, int ACCESS>
static void run_encode(const void* x, int64_t ldx, int64_t m, int64_t d, const Codes& out, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(m * out.groups, kWarps * kAhead));
  if constexpr (ACCESS == 4 * (int)sizeof(T)) {
    if (d % kGroup == 0) {
      launch_dependent(encode_kernel<T, ACCESS, true>, grid, kThreads, 0, st, (const T*)x, ldx, m, (int)d, out);
      return;
    }
  }
  launch_dependent(encode_kernel<T, ACCESS, false>, grid, kThreads, 0, st, (const T*)x, ldx, m, (int)d, out);
}
template <typename T, int ACCESS>
static void run_values(const Codes& in, void* out, int64_t ldo, int64_t m, int64_t d, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(m * in.groups, kWarps * kAhead));
  launch_dependent(values_kernel<T, ACCESS>, grid, kThreads, 0, st, in, (T*)out, ldo, m, (int)d);
}

}  // namespace ckpt
}  // namespace f2c

using namespace f2c;
using namespace f2c::ckpt;

extern "C" int f2c_checkpoint_int8(const void* x, int64_t ldx, int dtype, int64_t m, int64_t d, uint8_t* codes, int64_t ldq, float* scales, void* stream) {
  const char* op = "checkpoint_int8";
  if (const int rc = check_sizes(op, dtype, m, d)) return rc;
  if (const int rc = check_codes(op, codes, ldq, scales, m, d)) return rc;
  if (m == 0 || d == 0) return F2C_OK;
  F2C_REQUIRE(x, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(m == 1 || ldx >= d, F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  const Codes out{codes, ldq, scales, ceil_div(d, kGroup)};
  F2C_REQUIRE(m * out.groups <= kMaxRows, F2C_ERR_LIMIT, "%s: more than 2^31 groups", op);
  const int access = access_of(x, ldx, m, d, dtype_size(dtype));
  F2C_BY_ROWS(run_encode, dtype, access, x, ldx, m, d, out, (cudaStream_t)stream);
  return check_launch(op);
}

extern "C" int f2c_checkpoint_values(const uint8_t* codes, int64_t ldq, const float* scales, int64_t m, int64_t d, void* out, int64_t ldo, int out_dtype,
                                     void* stream) {
  const char* op = "checkpoint_values";
  if (const int rc = check_sizes(op, out_dtype, m, d)) return rc;
  if (const int rc = check_codes(op, codes, ldq, scales, m, d)) return rc;
  if (m == 0 || d == 0) return F2C_OK;
  F2C_REQUIRE(out, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(m == 1 || ldo >= d, F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  const Codes in{const_cast<uint8_t*>(codes), ldq, const_cast<float*>(scales), ceil_div(d, kGroup)};
  F2C_REQUIRE(m * in.groups <= kMaxRows, F2C_ERR_LIMIT, "%s: more than 2^31 groups", op);
  const int access = access_of(out, ldo, m, d, dtype_size(out_dtype));
  F2C_BY_ROWS(run_values, out_dtype, access, in, out, ldo, m, d, (cudaStream_t)stream);
  return check_launch(op);
}
