// What the 8-bit products share between their files (int8_quantize.cu, int8_mm.cu, int8_few.cu, int8_linear.cu).
#pragma once
#include "tcgen05.cuh"

namespace f2c {
namespace i8 {

using namespace t5;

constexpr int kMaxK = 131071;                 // 128 * 128 * k stays below 2^31: the int32 sum is exact
constexpr int64_t kMaxRows = (1ll << 31) - 4096;
constexpr int kM = 128, kK = 128, kMaxN = 256;
constexpr int kABytes = kM * kK;

// Rows in floating point: the columns of x1, then those of x2.
struct Rows {
  const void *x1, *x2;
  int64_t ld1, ld2, k1, k2, m;
  int dtype;
  // whether their starts and lengths, and those of their codes, allow reads of `bytes`
  bool fits(int bytes, const int8_t* codes, int64_t ldq) const {
    const int64_t v = bytes / dtype_size(dtype);
    return aligned(x1, bytes) && aligned(x2, bytes) && aligned(codes, v) && k1 % v == 0 && k2 % v == 0 && (m <= 1 || (ld1 % v == 0 && ld2 % v == 0 && ldq % v == 0));
  }
};

int check_rows(const char* op, const Rows& r);
int quantize(const Rows& r, int8_t* codes, int64_t ldq, float* scales, cudaStream_t st);

static int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }
static int64_t round16(int64_t v) { return (v + 15) / 16 * 16; }
static bool in_place(const int8_t* p, int64_t ld, int64_t rows) { return aligned(p, 16) && (rows <= 1 || ld % 16 == 0); }

struct Operand {
  const int8_t* p;
  int64_t ld, rows;
};

struct Plan {
  int channel_tiles, tile_rows, items, steps, split, stages;
  int ctas;  // that share a tile's channels: 1, or 2 with twice as many
  int parts_at, share_log;
  int tmem, accumulators;  // columns of one accumulator: a power of two; and how many, two where a CTA has more than one tile
  unsigned grid;
  size_t smem;
};

struct Job {
  Operand a, b;
  const float *a_scales, *b_scales, *bias;
  void* out;
  int64_t k;
  int relu, out_dtype, weights_first;
  uint32_t tries;  // of the kernels' bounded waits
  void activation(int flags) {  // relu, or with F2C_NO_WAITS
    relu = (flags & ~F2C_NO_WAITS) != 0;
    tries = flags & F2C_NO_WAITS ? 0u : kWaitLimit;
  }
};

int check(const char* op, int64_t m, int64_t n, int64_t k, int out_dtype);
Plan plan(int64_t m, int64_t n, int64_t k, int sms);
// The operand where TMA can read it: its own memory, or a copy in the workspace (which moves on).
Operand readable(const Operand& o, int64_t k, char*& ws, cudaStream_t st);
int mm(const char* op, const Job& j, cudaStream_t st);
// The kernel for little work (int8_few.cu): whether it is the faster one, whether it encodes rows in floating point on the way, and itself (rows of
// codes have dtype I8 and j.a_scales).
bool is_few(int64_t m, int64_t n, int64_t k);
bool few_encodes(const Rows& x, int64_t n);
int few(const char* op, const Rows& x, const Job& j, cudaStream_t st);

// ---------------------------------------------------------------- codes
struct Scale {
  float scale, inv;  // inv 0: divide
  bool zero;         // all codes are
};
// of the bits of a row's largest magnitude: those of infinities and NaNs are larger than all others
__device__ __forceinline__ Scale scale_of(uint32_t largest) {
  const bool bad = largest >= 0x7f800000u;
  Scale s;
  s.scale = bad ? __int_as_float(0x7fffffff) : __fdiv_rn(__uint_as_float(largest), 127.0f);
  s.zero = bad || s.scale == 0.0f;
  s.inv = s.zero || s.scale < 1e-37f ? 0.0f : __frcp_rn(s.scale);  // (the reciprocal of less has no place, or few bits)
  return s;
}

// The codes of N (up to 4) values, one in a byte.  One branch for all of them: a branch for each made a warp wait out four chains of
// dependent instructions one after the other (5003 rows of 602 float16: 10.2 us, and 5.6 with one).
template <int N>
__device__ __forceinline__ uint32_t codes_of(const float (&v)[N], const Scale& s) {
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to even and leaves the integer in the low bits
  uint32_t code[4] = {};
  float far = 0.0f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float t = v[e] * s.inv, shifted = t + kRound;
    far = fmaxf(far, fabsf(t - (shifted - kRound)));
    code[e] = __float_as_uint(shifted);
  }
  if (s.inv == 0.0f || far > 0.4999f) {
#pragma unroll
    for (int e = 0; e < N; ++e) code[e] = __float_as_uint(fminf(fmaxf(rintf(__fdiv_rn(v[e], s.scale)), -127.0f), 127.0f) + kRound);
  }
  const uint32_t word = __byte_perm(__byte_perm(code[0], code[1], 0x0040), __byte_perm(code[2], code[3], 0x0040), 0x5410);
  return s.zero ? 0u : word;
}

// The largest magnitude of values in 32-bit words (two of a 16-bit type), by their bits.
template <typename T>
struct Largest {
  uint32_t bits = 0u;
  __device__ __forceinline__ void add(uint32_t word) { bits = sizeof(T) == 4 ? max(bits, word & 0x7fffffffu) : __vmaxu2(bits, word & 0x7fff7fffu); }
  __device__ __forceinline__ uint32_t of_float() const {
    if constexpr (sizeof(T) == 4) return bits;
    union { uint16_t u; T t; } h;
    h.u = (uint16_t)max(bits >> 16, bits & 0xffffu);
    return __float_as_uint(to_float(h.t));
  }
};

template <int BYTES> struct Words;  // a vector of BYTES
template <> struct Words<16> { using type = uint4; };
template <> struct Words<8> { using type = uint2; };
template <> struct Words<4> { using type = uint32_t; };
template <> struct Words<2> { using type = uint16_t; };

template <typename T, int BYTES>
struct Vector {
  static constexpr int V = BYTES / (int)sizeof(T), W = BYTES < 4 ? 1 : BYTES / 4;
  static constexpr int G = V < 4 ? 4 / V : 1;  // vectors that are encoded together: four values share a branch
  union { typename Words<BYTES>::type raw; uint32_t w[W]; T v[V]; };
  __device__ __forceinline__ Vector() {
#pragma unroll
    for (int e = 0; e < W; ++e) w[e] = 0u;
  }
};

// The codes of G vectors to their places, `step` bytes apart; the first `count` of them.
template <typename T, int BYTES>
__device__ __forceinline__ void write(int8_t* to, int step, int count, const Vector<T, BYTES>* v, const Scale& s) {
  constexpr int V = Vector<T, BYTES>::V, G = Vector<T, BYTES>::G;
  if constexpr (G == 1) {
    uint32_t word[V / 4];
#pragma unroll
    for (int g = 0; g < V; g += 4) {
      const float f[4] = {to_float(v->v[g]), to_float(v->v[g + 1]), to_float(v->v[g + 2]), to_float(v->v[g + 3])};
      word[g / 4] = codes_of(f, s);
    }
    if (count > 0) {
      if constexpr (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(word[0], word[1]);
      else *reinterpret_cast<uint32_t*>(to) = word[0];
    }
  } else {
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = to_float(v[e / V].v[e % V]);
    const uint32_t word = codes_of(f, s);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (g >= count) break;
      if constexpr (V == 2) *reinterpret_cast<uint16_t*>(to + g * step) = (uint16_t)(word >> (16 * g));
      else to[g * step] = (int8_t)(word >> (8 * g));
    }
  }
}

// ---------------------------------------------------------------- results
// scale * sum + bias, not below `floor`; a NaN stays one
__device__ __forceinline__ float finish(int sum, float scale, float bias, float floor) {
  const float v = fmaf((float)sum, scale, bias);
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(floor));
  return r;
}

// One channel of 32 rows of out, `rows` of which exist.
template <typename T>
__device__ __forceinline__ void store_rows(T* out, int64_t ld, const uint32_t (&r)[32], const float* row_scale, float w_scale, float bias, float floor, int rows) {
  if (rows >= 32) {
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 s = *reinterpret_cast<const float4*>(row_scale + j);
      const float of[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int e = 0; e < 4; ++e, out += ld) *out = from_float<T>(finish((int)r[j + e], of[e] * w_scale, bias, floor));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j, out += ld)
      if (j < rows) *out = from_float<T>(finish((int)r[j], row_scale[j] * w_scale, bias, floor));
  }
}

}  // namespace i8
}  // namespace f2c
