// Rows four columns a lane (layer_norm.cu, layer_norm_backward.cu, checkpoint.cu), and activations in 8 bits:
// of every row, 128 columns at a time - four of each lane of a warp - are a group with codes 0 .. 255,
//   low = min,  step = (max - low) / 255,  code = round-to-even((x - low) / step),  value = low + step * code,
// the differences and quotients as single precision has them, so that every implementation of the definition gives the same codes.
// A group whose max - low is not finite (it holds a NaN or an infinity, or more than the type's range) has codes 0 and values NaN.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace f2c {
namespace ckpt {

constexpr int kGroup = F2C_CHECKPOINT_GROUP;  // columns of a warp, four a lane
static_assert(kGroup == 128, "a group is what a warp holds");
constexpr int64_t kMaxRows = 1ll << 31, kMaxColumns = 1 << 20;

// Two single-precision numbers in a register pair, and what is done to both by one instruction (add2, lo32 and hi32: common.cuh).
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair_of(float x, float y) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 both(float v) { return pair_of(v, v); }
__device__ __forceinline__ f32x2 plus2(f32x2 a, f32x2 b) {
  add2(a, b);
  return a;
}

// 0 without a load when !on; no branch.  (Narrow loads of neighbouring lanes share sectors: they may stay in L1.)
__device__ __forceinline__ uint2 ld_u64_if(const void* p, bool on) {
  uint2 v = make_uint2(0u, 0u);
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %3, 0;\n\t@q ld.global.nc.v2.u32 {%0,%1}, [%2];\n\t}" : "+r"(v.x), "+r"(v.y) : "l"(p), "r"((uint32_t)on));
  return v;
}
__device__ __forceinline__ uint32_t ld_u32_if(const void* p, bool on) {
  uint32_t v = 0u;
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q ld.global.nc.u32 %0, [%1];\n\t}" : "+r"(v) : "l"(p), "r"((uint32_t)on));
  return v;
}
__device__ __forceinline__ uint16_t ld_u16_if(const void* p, bool on) {
  uint16_t v = 0;
  asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t@q ld.global.nc.u16 %0, [%1];\n\t}" : "+h"(v) : "l"(p), "r"((uint32_t)on));
  return v;
}

// Four columns of a row as they are in memory.  ACCESS: bytes of a load or store, by what the rows' alignment and length allow.
template <typename T, int ACCESS>
struct alignas(4 * sizeof(T)) Four {
  static constexpr int kEach = ACCESS / (int)sizeof(T), kPieces = 4 / kEach;
  T v[4];

  // the row's columns from `at` on, of which `left` (which may be negative) exist; zeros for the others
  __device__ __forceinline__ void load(const T* at, int left) {
    if constexpr (ACCESS == 16) {
      const uint4 w = ldg_nc_u128_if(at, left > 0);
      *reinterpret_cast<uint4*>(v) = w;
    } else if constexpr (kPieces == 1) {
      *reinterpret_cast<uint2*>(v) = ldg_nc_u64_if(at, left > 0);
    } else {
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const bool here = p * kEach < left;
        if constexpr (ACCESS == 8) *reinterpret_cast<uint2*>(v + p * kEach) = ld_u64_if(at + p * kEach, here);
        else if constexpr (ACCESS == 4) *reinterpret_cast<uint32_t*>(v + p * kEach) = ld_u32_if(at + p * kEach, here);
        else *reinterpret_cast<uint16_t*>(v + p) = ld_u16_if(at + p, here);
      }
    }
  }
  __device__ __forceinline__ void store(T* at, int left) const {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      if (p * kEach >= left) continue;
      if constexpr (ACCESS == 16) *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(v);
      else if constexpr (ACCESS == 8) *reinterpret_cast<uint2*>(at + p * kEach) = *reinterpret_cast<const uint2*>(v + p * kEach);
      else if constexpr (ACCESS == 4) *reinterpret_cast<uint32_t*>(at + p * kEach) = *reinterpret_cast<const uint32_t*>(v + p * kEach);
      else at[p] = v[p];
    }
  }
  __device__ __forceinline__ void get(f32x2 (&f)[2]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) f[h] = pair_of(to_float(v[2 * h]), to_float(v[2 * h + 1]));
  }
  __device__ __forceinline__ void set(const f32x2 (&f)[2]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v[2 * h] = lo32(f[h]);
        v[2 * h + 1] = hi32(f[h]);
      }
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<__half2*>(v + 2 * h) = __floats2half2_rn(lo32(f[h]), hi32(f[h]));
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<__nv_bfloat162*>(v + 2 * h) = __floats2bfloat162_rn(lo32(f[h]), hi32(f[h]));
    }
  }
};

// Bytes of an access that rows of `item`-byte elements starting at `p`, `ld` elements apart and d long, allow; at most four elements.
static inline int access_of(const void* p, int64_t ld, int64_t m, int64_t d, int item) {
  int a = 4 * item;
  while (a > item && (!aligned(p, a) || d * item % a != 0 || (m > 1 && ld * item % a != 0))) a /= 2;
  return a;
}

// of two or three, NaN where one is
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float warp_min_nan(float v) {
  float r;
  asm volatile("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

struct Scale { float step, low; };

// Codes of four columns of which `left` exist, by divisions.
static __device__ __noinline__ uint32_t encode_by_division(float x0, float x1, float x2, float x3, float low, float step, int left) {
  const float x[4] = {x0, x1, x2, x3};
  uint32_t codes = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) codes |= (uint32_t)fminf(rintf((x[e] - low) / step), 255.0f) << (8 * e);
  return codes;
}

// A group's extremes, four columns a lane of which `left` exist: by whole warps, all lanes get them.  Columns that are not there get the first one's value.
struct Extremes { float low, high; };
__device__ __forceinline__ Extremes extremes_of(f32x2 (&x)[2], int left) {
  float low = min_nan(min_nan(lo32(x[0]), hi32(x[0]), lo32(x[1])), hi32(x[1])), high = max_nan(max_nan(lo32(x[0]), hi32(x[0]), lo32(x[1])), hi32(x[1]));
  if (left < 4) {
    const float first = lo32(x[0]);
    const float second = left > 1 ? hi32(x[0]) : first, third = left > 2 ? lo32(x[1]) : first;
    x[0] = pair_of(first, second);
    x[1] = pair_of(third, first);
    low = left > 0 ? min_nan(first, second, third) : __int_as_float(0x7f800000);  // (without any: nobody's extreme)
    high = left > 0 ? max_nan(first, second, third) : __int_as_float(0xff800000);
  }
  return Extremes{warp_min_nan(low), warp_max_nan(high)};
}

// Step and lowest value, the step's reciprocal, and whether the quotients are to be had with it (not where the range is so small or so large that remainders
// would not be exact, or is none).
struct Steps {
  Scale s;
  float by;
  bool plain;
};
__device__ __forceinline__ Steps steps_of(Extremes e) {
  Steps r;
  const float range = e.high - e.low;
  r.s.low = e.low;
  r.s.step = div_exact_fast(range, 255.0f, 1.0f / 255.0f);  // two corrections with exact remainders
  r.by = __frcp_rn(r.s.step);
  r.plain = range > 1e-25f && range < 1e30f;
  if (!r.plain) {
    const bool none = !(range <= 3.402823466e38f);  // infinite, or no number
    r.s.step = none ? __int_as_float(0x7fffffff) : range / 255.0f;
    if (none) r.s.low = r.s.step;
  }
  return r;
}

// The codes of a lane's four columns (0 for those that are not there).  The quotients are what division gives: the product with the correctly rounded reciprocal, and two
// corrections with exact remainders (Markstein).  (Corrected only where the product lay near a tie: rows of 16-bit numbers, whose quotients are ties as often as
// not somewhere in a group, took twice the time.)  2^23 + 2^22 added to a number below 2^22 rounds it to even and leaves it in the last bits.
__device__ __forceinline__ uint32_t codes_of(const f32x2 (&x)[2], int left, Scale s, float reciprocal, bool plain) {
  if (!plain) {
    if (!(s.step > 0.0f)) return 0u;
    return encode_by_division(lo32(x[0]), hi32(x[0]), lo32(x[1]), hi32(x[1]), s.low, s.step, left);
  }
  const f32x2 by = both(reciprocal), less = both(-s.low), minus = both(-s.step), magic = both(12582912.0f);
  f32x2 m[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const f32x2 over = plus2(x[h], less);
    f32x2 q = mul2(over, by);
    q = fma2(fma2(q, minus, over), by, q);
    q = fma2(fma2(q, minus, over), by, q);
    m[h] = plus2(q, magic);
  }
  const uint32_t codes = __byte_perm(__byte_perm((uint32_t)m[0], (uint32_t)(m[0] >> 32), 0x0040), __byte_perm((uint32_t)m[1], (uint32_t)(m[1] >> 32), 0x0040), 0x5410);
  return left >= 4 ? codes : left <= 0 ? 0u : codes & ((1u << (8 * left)) - 1u);
}

// Codes and scale of a group; by whole warps.
__device__ __forceinline__ uint32_t encode(const f32x2 (&given)[2], int left, Scale& s) {
  f32x2 x[2] = {given[0], given[1]};
  const Steps r = steps_of(extremes_of(x, left));
  s = r.s;
  return codes_of(x, left, r.s, r.by, r.plain);
}

// The codes as numbers: 2^23 + q, and -2^23 (or another number that leaves whole ones).
__device__ __forceinline__ void numbers_of(uint32_t codes, f32x2 less, f32x2 (&q)[2]) {
  q[0] = plus2(pair_of(__uint_as_float(__byte_perm(codes, 0x4B000000u, 0x7440)), __uint_as_float(__byte_perm(codes, 0x4B000000u, 0x7441))), less);
  q[1] = plus2(pair_of(__uint_as_float(__byte_perm(codes, 0x4B000000u, 0x7442)), __uint_as_float(__byte_perm(codes, 0x4B000000u, 0x7443))), less);
}
__device__ __forceinline__ void decode(uint32_t codes, Scale s, f32x2 (&x)[2]) {
  numbers_of(codes, both(-8388608.0f), x);
#pragma unroll
  for (int h = 0; h < 2; ++h) x[h] = fma2(both(s.step), x[h], both(s.low));
}

__device__ __forceinline__ Scale load_scale(const float* at) {
  const float2 v = __ldg(reinterpret_cast<const float2*>(at));
  return Scale{v.x, v.y};
}
__device__ __forceinline__ void store_scale(float* at, Scale s) { *reinterpret_cast<float2*>(at) = make_float2(s.step, s.low); }

// Codes, their row stride in bytes, and [rows][groups][step, low].
struct Codes {
  uint8_t* codes;
  int64_t ld;
  float* scales;
  int64_t groups;
};

// What the entry points refuse of codes: rows start on 16 bytes, with room for whole 16 bytes, and scales on 8.
int check_codes(const char* op, const uint8_t* codes, int64_t ldq, const float* scales, int64_t m, int64_t d);
int check_sizes(const char* op, int dtype, int64_t m, int64_t d);

}  // namespace ckpt
}  // namespace f2c

// a type and an access width as template arguments
#define F2C_BY_ROWS(run, dtype, access, ...)                                   \
  do {                                                                         \
    if (dtype == F2C_F32) {                                                    \
      if (access == 16) run<float, 16>(__VA_ARGS__);                           \
      else if (access == 8) run<float, 8>(__VA_ARGS__);                        \
      else run<float, 4>(__VA_ARGS__);                                         \
    } else if (dtype == F2C_F16) {                                             \
      if (access == 8) run<__half, 8>(__VA_ARGS__);                            \
      else if (access == 4) run<__half, 4>(__VA_ARGS__);                       \
      else run<__half, 2>(__VA_ARGS__);                                        \
    } else {                                                                   \
      if (access == 8) run<__nv_bfloat16, 8>(__VA_ARGS__);                     \
      else if (access == 4) run<__nv_bfloat16, 4>(__VA_ARGS__);                \
      else run<__nv_bfloat16, 2>(__VA_ARGS__);                                 \
    }                                                                          \
  } while (0)
