// The 8-bit product for little work, where int8_mm.cu's way through TMA, shared memory and TMEM is longer than the work.
//
// A CTA has 16 rows and 16 to 128 channels; its eight warps share out channels (16 each) and parts of K, whose sums they add in shared
// memory.  A lane reads 16 neighbouring columns of a channel straight into registers, so that all of a warp's weights are on their way at
// once.  The rows' codes are put into shared memory, or made there: then a warp has two rows, finds their largest magnitudes and encodes them.
// The sums are four-element dot products, 256 products a cycle and SM; the warp-wide 8-bit MMA has about 25 here (16 x 4096 x 4096: 17.7 us with
// it).  What bounds it is latency: launch, loads, sums (1 x 172 x 256: 2.8 us).
#include "int8_mm.cuh"

namespace f2c {
namespace i8f {

using namespace i8;

constexpr int kWarps = 8, kThreads = 32 * kWarps, kRows = 16, kGroups = 2, kUnit = 64;  // columns of K that a warp takes at a time
constexpr int kAhead = 4;    // units in flight
constexpr int kKept = 4;     // vectors of a row that a lane keeps
constexpr int kMaxCodes = 2048;  // columns of rows that are encoded here

struct Params {
  Rows x;
  const int8_t* w;
  int64_t ldw;
  const float *a_scales, *b_scales, *bias;
  void* out;
  int n, k, relu;
  int k_parts;            // warps that share a channel's K
};

// 16 columns from t on of a row of a matrix whose last byte is in front of `end`; zeros behind the row
__device__ __forceinline__ uint4 read16(const int8_t* row, int t, int k, const int8_t* end) {
  uint4 v = make_uint4(0u, 0u, 0u, 0u);
  if (t + 16 <= k || (t < k && row + t + 16 <= end)) {
    v = __ldg(reinterpret_cast<const uint4*>(row + t));  // what comes behind the row meets codes of zero
  } else if (t < k) {
    uint32_t w[4] = {};
    for (int e = 0; t + e < k; ++e) w[e >> 2] |= (uint32_t)(uint8_t)__ldg(row + t + e) << (8 * (e & 3));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}

// the first n bytes of 16
__device__ __forceinline__ uint4 first_bytes(uint4 v, int n) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int left = n - 4 * e;
    w[e] = left <= 0 ? 0u : left < 4 ? w[e] & ((1u << (8 * left)) - 1u) : w[e];
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// T: what the rows are, int8_t for codes; BYTES of it are read at a time
template <typename T, typename O, int BYTES>
__global__ void __launch_bounds__(kThreads, 2) few_kernel(const Params p) {
  constexpr bool kEncodes = sizeof(T) > 1;
  extern __shared__ __align__(16) int8_t codes_s[];  // [row][pitch]
  __shared__ int sums_s[kWarps][kRows][8 * kGroups];
  __shared__ float scale_s[kRows];
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  const int part = wid % p.k_parts, column = wid / p.k_parts, columns = kWarps / p.k_parts;
  const int64_t row0 = (int64_t)blockIdx.x * kRows;
  const int rows = (int)min((int64_t)kRows, p.x.m - row0), channel0 = ((int)blockIdx.y * columns + column) * 8 * kGroups;
  const int units = (p.k + kUnit - 1) / kUnit, at = (lane & 3) * 16;
  const int8_t* const end = p.w + (int64_t)(p.n - 1) * p.ldw + p.k;
  const int8_t* w[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) w[g] = p.w + (int64_t)min(channel0 + 8 * g + (lane >> 2), p.n - 1) * p.ldw;

  uint4 b[kAhead][kGroups];
  auto weights = [&](int u, uint4 (&to)[kGroups]) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) to[g] = u < units ? read16(w[g], u * kUnit + at, p.k, end) : make_uint4(0u, 0u, 0u, 0u);
  };
  dependency_wait();
#pragma unroll
  for (int q = 0; q < kAhead; ++q) weights(part + q * p.k_parts, b[q]);
  release_dependents();

  const int pitch = units * kUnit + 64;  // rows that follow one another start in different halves of the banks
  if constexpr (kEncodes) {
    using Vec = Vector<T, BYTES>;
    using R = typename Words<BYTES>::type;
    constexpr int V = Vec::V;
    const int n1 = (int)(p.x.k1 / V), n = n1 + (int)(p.x.k2 / V);
    const R* x1[2];
    const R* x2[2];
    Vec kept[2][kKept];
    Largest<T> largest[2];
    auto read = [&](int i, int v) {
      Vec r;
      r.raw = __ldg(v < n1 ? x1[i] + v : x2[i] + v);
      return r;
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = wid + i * kWarps;
      x1[i] = reinterpret_cast<const R*>((const T*)p.x.x1 + (row0 + r) * p.x.ld1);
      x2[i] = reinterpret_cast<const R*>((const T*)p.x.x2 + (row0 + r) * p.x.ld2) - n1;
      if (r >= rows) continue;
#pragma unroll
      for (int q = 0; q < kKept; ++q)
        if (lane + 32 * q < n) kept[i][q] = read(i, lane + 32 * q);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = wid + i * kWarps;
      if (r >= rows) continue;
      auto look = [&](const Vec& v) {
#pragma unroll
        for (int e = 0; e < Vec::W; ++e) largest[i].add(v.w[e]);
      };
#pragma unroll
      for (int q = 0; q < kKept; ++q) look(kept[i][q]);
      for (int v = lane + 32 * kKept; v < n; v += 32) look(read(i, v));
      const Scale s = scale_of(__reduce_max_sync(0xffffffffu, largest[i].of_float()));
      if (lane == 0) scale_s[r] = s.scale;
      int8_t* to = codes_s + r * pitch;
      const auto some = [&](int v) { return v < n ? (n - v + 31) / 32 : 0; };
#pragma unroll
      for (int q = 0; q < kKept; q += Vec::G)
        if (lane + 32 * q < n) write<T, BYTES>(to + (lane + 32 * q) * V, 32 * V, some(lane + 32 * q), kept[i] + q, s);
      for (int v = lane + 32 * kKept; v < n; v += 32 * Vec::G) {
        Vec x[Vec::G];
#pragma unroll
        for (int g = 0; g < Vec::G; ++g)
          if (v + 32 * g < n) x[g] = read(i, v + 32 * g);
        write<T, BYTES>(to + v * V, 32 * V, some(v), x, s);
      }
      for (int t = p.k + lane; t < units * kUnit; t += 32) to[t] = 0;
    }
    __syncthreads();
  } else {
    const int8_t* const rows_end = (const int8_t*)p.x.x1 + (p.x.m - 1) * p.x.ld1 + p.k;
    const int chunks = units * (kUnit / 16);
    for (int i = tid; i < rows * chunks; i += kThreads) {
      const int r = i / chunks, t = i % chunks * 16;
      *reinterpret_cast<uint4*>(codes_s + r * pitch + t) = first_bytes(read16((const int8_t*)p.x.x1 + (row0 + r) * p.x.ld1, t, p.k, rows_end), p.k - t);
    }
    if (tid < rows) scale_s[tid] = __ldg(p.a_scales + row0 + tid);
    __syncthreads();
  }

  int d[kGroups][kRows] = {};
  for (int u0 = part; u0 < units; u0 += kAhead * p.k_parts) {
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int u = u0 + q * p.k_parts;
      if (u >= units) break;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (r >= rows) break;
        const uint4 x = *reinterpret_cast<const uint4*>(codes_s + r * pitch + u * kUnit + at);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          d[g][r] = __dp4a((int)x.x, (int)b[q][g].x, d[g][r]);
          d[g][r] = __dp4a((int)x.y, (int)b[q][g].y, d[g][r]);
          d[g][r] = __dp4a((int)x.z, (int)b[q][g].z, d[g][r]);
          d[g][r] = __dp4a((int)x.w, (int)b[q][g].w, d[g][r]);
        }
      }
      weights(u + kAhead * p.k_parts, b[q]);
    }
  }
  // four lanes have a channel
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    if (r >= rows) break;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      int v = d[g][r];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if ((lane & 3) == 0) sums_s[wid][r][8 * g + (lane >> 2)] = v;
    }
  }
  __syncthreads();
  // thread = channel of the CTA, and every so manieth row
  const int width = columns * 8 * kGroups, c = tid % width, channel = (int)blockIdx.y * width + c;
  if (channel < p.n) {
    const float w_scale = __ldg(p.b_scales + channel), bias = p.bias != nullptr ? __ldg(p.bias + channel) : 0.0f;
    const float floor = p.relu ? 0.0f : __int_as_float(0xff800000);
    const int warp = c / (8 * kGroups) * p.k_parts, in = c % (8 * kGroups);
    for (int r = tid / width; r < rows; r += kThreads / width) {
      int sum = 0;
      for (int q = 0; q < p.k_parts; ++q) sum += sums_s[warp + q][r][in];
      ((O*)p.out)[(row0 + r) * p.n + channel] = from_float<O>(finish(sum, scale_s[r] * w_scale, bias, floor));
    }
  }
}

template <typename T, typename O>
static cudaError_t by_width(const Params& p, dim3 grid, size_t smem, cudaStream_t st) {
  if constexpr (sizeof(T) == 1) {
    return launch_dependent(few_kernel<T, O, 16>, grid, kThreads, smem, st, p);
  } else {
    if (p.x.fits(16, nullptr, 0)) return launch_dependent(few_kernel<T, O, 16>, grid, kThreads, smem, st, p);
    if constexpr (sizeof(T) == 2) {
      if (!p.x.fits(4, nullptr, 0)) return launch_dependent(few_kernel<T, O, 2>, grid, kThreads, smem, st, p);
    }
    return launch_dependent(few_kernel<T, O, 4>, grid, kThreads, smem, st, p);
  }
}

template <typename T>
static cudaError_t by_output(int out_dtype, const Params& p, dim3 grid, size_t smem, cudaStream_t st) {
  if (out_dtype == F2C_F32) return by_width<T, float>(p, grid, smem, st);
  if (out_dtype == F2C_F16) return by_width<T, __half>(p, grid, smem, st);
  return by_width<T, __nv_bfloat16>(p, grid, smem, st);
}

// Warps that share a channel's K: as few as leave every SM a CTA and a warp no more than kAhead units.
static int k_parts(int64_t m, int64_t n, int64_t k) {
  const int64_t row_tiles = ceil_div(m, kRows), units = ceil_div(k, kUnit);
  int parts = 1;
  while (parts < kWarps && parts < units && (row_tiles * ceil_div(n, kWarps / parts * 8 * kGroups) < current_sm_count() * 3 / 4 || parts * 4 * kAhead < units))
    parts *= 2;
  return parts;
}

}  // namespace i8f

namespace i8 {

// Codes in hand: 1 x 172 x 256 2.6 us here and 3.4 there, 1 x 4096 x 2048 4.9 and 6.2, 4 x 4096 x 2048 6.3 and 6.4, 16 x 172 x 256 3.8 and 3.7.
bool is_few(int64_t m, int64_t n, int64_t k) { return m <= 4 && k > 0 && k <= i8f::kMaxCodes; }

// Every CTA encodes its rows again, which saves a launch: 16 x 172 x 256 and 16 x 1024 x 1024 are even without the encoding.
bool few_encodes(const Rows& x, int64_t n) {
  const int64_t k = x.k1 + x.k2;
  return is_few(x.m, n, k) || (x.m <= 16 && k > 0 && k <= i8f::kMaxCodes && n * k <= (1 << 20));
}

int few(const char* op, const Rows& x, const Job& j, cudaStream_t st) {
  const int64_t k = j.k, n = j.b.rows;
  i8f::Params p{x, j.b.p, j.b.ld, j.a_scales, j.b_scales, j.bias, j.out, (int)n, (int)k, j.relu, i8f::k_parts(x.m, n, k)};
  const dim3 grid((unsigned)ceil_div(x.m, i8f::kRows), (unsigned)ceil_div(n, i8f::kWarps / p.k_parts * 8 * i8f::kGroups));
  const size_t smem = (size_t)i8f::kRows * (ceil_div(k, i8f::kUnit) * i8f::kUnit + 64);
  const cudaError_t e = x.dtype == F2C_I8    ? i8f::by_output<int8_t>(j.out_dtype, p, grid, smem, st)
                        : x.dtype == F2C_F32 ? i8f::by_output<float>(j.out_dtype, p, grid, smem, st)
                        : x.dtype == F2C_F16 ? i8f::by_output<__half>(j.out_dtype, p, grid, smem, st)
                                             : i8f::by_output<__nv_bfloat16>(j.out_dtype, p, grid, smem, st);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return set_error(F2C_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
  }
  return check_launch(op);
}

}  // namespace i8
}  // namespace f2c
