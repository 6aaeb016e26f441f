// act(x w^T + b) with x quantised on the way (f2c_int8_linear): one kernel where there is little of x in a tile of the product, otherwise
// f2c_int8_quantize and f2c_int8_mm one after the other.
//
// The one kernel has int8_mm.cu's tiles (128 channels x up to 64 rows), one to a CTA, and makes their right operand itself: while TMA brings all
// of the tile's weights, a warp has two or four rows in registers, finds their largest magnitudes and writes their codes where the MMAs read them (128-byte
// swizzle).  CTAs with the same rows and other channels encode them again.  It saves a launch, which is what the call waits for there: 1024 x 172 x 256
// takes the host 7.0 us in two launches.  What bounds it is the chain of rows, codes, MMAs and results, 4.5 us of the device there.
#include "int8_mm.cuh"

namespace f2c {
namespace i8l {

using namespace i8;

constexpr int kWarps = 8, kThreads = 64 + 32 * kWarps;  // warp 0: TMA, warp 1: MMA, then those that encode and write
constexpr int kMaxSteps = 8, kMaxRows = 64, kMaxEncoded = 16 * 1024;  // of K; rows of a tile; elements of x that a CTA encodes

struct Params {
  Rows x;
  const float *b_scales, *bias;
  void* out;
  int n, steps, channel_tiles, tile_rows, tmem, relu;
  uint32_t tries;  // of a role's bounded waits; 0: nothing is issued
  int* error;
};

struct Bars {
  uint64_t full[kMaxSteps], codes, acc, drain;
  uint32_t tmem;
  int failed;
};

__device__ __forceinline__ void barrier_of_warps() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }

// T: the rows' type, of which BYTES are read at a time; a lane keeps KEPT vectors of ROWS rows
template <typename T, typename O, int BYTES, int ROWS, int KEPT>
__global__ void __launch_bounds__(kThreads, 2) linear_kernel(const __grid_constant__ CUtensorMap w, const Params p) {
  using Vec = Vector<T, BYTES>;
  using R = typename Words<BYTES>::type;
  constexpr int V = Vec::V;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Bars bars;
  __shared__ __align__(16) float scale_s[kMaxRows];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  const int channel0 = (int)blockIdx.x % p.channel_tiles * kM;
  const int64_t row0 = (int64_t)((int)blockIdx.x / p.channel_tiles) * p.tile_rows;
  const int rows = (int)min((int64_t)p.tile_rows, p.x.m - row0);
  const uint32_t b_bytes = (uint32_t)p.tile_rows * kK;
  unsigned char* codes = smem + (size_t)p.steps * kABytes;  // [step][row][128], behind the weights
  uint32_t left = p.tries;

  if (wid == 1) alloc_tmem(&bars.tmem, (uint32_t)p.tmem);
  if (tid == 0) {
    for (int i = 0; i < p.steps; ++i) init_bar(bars.full + i, 1);
    init_bar(&bars.codes, kWarps);
    init_bar(&bars.acc, 1);
    init_bar(&bars.drain, 1);
    fence_bars();
    bars.failed = 0;
    prefetch_map(&w);
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = bars.tmem;
  dependency_wait();
  if (wid == 0) {
    // ================= weights
    const bool mine = elected() != 0u && left != 0u;
    release_dependents();
    for (int i = 0; i < p.steps; ++i) {
      expect_if(mine, bars.full + i, kABytes);
      tma_load(mine, &w, smem_u32(smem) + (uint32_t)i * kABytes, smem_u32(bars.full + i), i * kK, channel0);
    }
  } else if (wid == 1) {
    // ================= MMAs
    const bool mine = elected() != 0u;
    const uint32_t idesc = instruction(kSumS32, kFormatS8, kM, (uint32_t)p.tile_rows);
    const uint32_t a_low = desc_low(smem_u32(smem), kChunkAlongK), b_low = desc_low(smem_u32(codes), kChunkAlongK);
    wait_bar(&bars.codes, 0, left);
    for (int i = 0; i < p.steps; ++i) {
      wait_bar(bars.full + i, 0, left);
      fence_after();
      const uint32_t a = a_low + (uint32_t)i * (kABytes >> 4), b = b_low + (uint32_t)i * (b_bytes >> 4);
#pragma unroll
      for (uint32_t q = 0; q < kK / 32; ++q) mma_i8(mine && left != 0u, tmem, desc(a + q * kStepAlongK), desc(b + q * kStepAlongK), idesc, i + (int)q != 0);
    }
    commit(mine && left != 0u, &bars.acc);
  } else {
    // ================= codes of the rows, then the results: a warp has the TMEM lanes of its quarter and every other 32 rows, thread = channel
    const int quarter = wid & 3, half = (wid - 2) >> 2, channel = channel0 + quarter * 32 + lane;
    const bool mine = channel < p.n;
    const float w_scale = mine ? __ldg(p.b_scales + channel) : 0.0f, bias = mine && p.bias != nullptr ? __ldg(p.bias + channel) : 0.0f;
    const int n1 = (int)(p.x.k1 / V), n = n1 + (int)(p.x.k2 / V);
    for (int r0 = (wid - 2) * ROWS; r0 < rows; r0 += kWarps * ROWS) {
      Vec kept[ROWS][KEPT];
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        if (r0 + i >= rows) break;
        const R* x1 = reinterpret_cast<const R*>((const T*)p.x.x1 + (row0 + r0 + i) * p.x.ld1);
        const R* x2 = reinterpret_cast<const R*>((const T*)p.x.x2 + (row0 + r0 + i) * p.x.ld2) - n1;
#pragma unroll
        for (int q = 0; q < KEPT; ++q) {
          const int v = lane + 32 * q;
          if (v < n) kept[i][q].raw = __ldg(v < n1 ? x1 + v : x2 + v);
        }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = r0 + i;
        if (r >= rows) break;
        Largest<T> largest;
#pragma unroll
        for (int q = 0; q < KEPT; ++q)
#pragma unroll
          for (int e = 0; e < Vec::W; ++e) largest.add(kept[i][q].w[e]);
        const Scale s = scale_of(__reduce_max_sync(0xffffffffu, largest.of_float()));
        if (lane == 0) scale_s[r] = s.scale;
        // column c of row r: step c / 128, its 16-byte pieces exchanged by the swizzle.  (Columns behind K meet weights of zero.)
#pragma unroll
        for (int q = 0; q < KEPT; ++q) {
          const int c = (lane + 32 * q) * V;
          if (lane + 32 * q < n)
            write<T, BYTES>(reinterpret_cast<int8_t*>(codes) + (size_t)(c / kK) * b_bytes + r * kK + ((((c & 127) >> 4) ^ (r & 7)) << 4) + (c & 15), 0, 1, &kept[i][q], s);
        }
      }
    }
    fence_async();
    __syncwarp();
    if (lane == 0) arrive(&bars.codes);
    barrier_of_warps();  // the rows' scales
    wait_bar(&bars.acc, 0, left);
    const bool lost = __any_sync(0xffffffffu, left == 0u);
    fence_after();
    for (int c0 = half * 32; c0 < rows; c0 += 64) {
      uint32_t r[32];
      tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c0, r);
      tmem_wait(r);
      if (mine)
        store_rows((O*)p.out + (row0 + c0) * p.n + channel, (int64_t)p.n, r, scale_s + c0, w_scale, lost ? __int_as_float(0x7fffffff) : bias,
                   p.relu ? 0.0f : __int_as_float(0xff800000), rows - c0);
      __syncwarp();
    }
  }
  if (left == 0u) bars.failed = 1;
  __syncwarp();
  fence_before();
  __syncthreads();
  if (bars.failed && p.tries != 0u) {
    // copies in flight write to shared memory, MMAs in flight read it and write TMEM: wait (bounded) for what was issued
    left = p.tries;
    if (wid == 0) {
      for (int i = 0; i < p.steps; ++i) wait_bar(bars.full + i, 0, left);
    } else if (wid == 1) {
      commit(elected() != 0u, &bars.drain);  // by who issued them
      wait_bar(&bars.drain, 0, left);
    }
    __syncthreads();
  }
  if (wid == 1) {
    fence_after();
    free_tmem(tmem, (uint32_t)p.tmem);
  }
  if (tid == 0 && bars.failed) report_wait(p.error, 7);
}

// bytes that are read at a time: four values or more, so that their codes are a word
static int width(const Rows& x) { return x.fits(16, nullptr, 0) ? 16 : dtype_size(x.dtype) == 2 && x.fits(8, nullptr, 0) ? 8 : 0; }

static bool one_launch(const Rows& x, const Plan& pl) {
  const int64_t k = x.k1 + x.k2;
  const int bytes = width(x);
  if (pl.steps < 1 || pl.steps > kMaxSteps || pl.split != 1 || pl.tile_rows > kMaxRows || pl.grid != (unsigned)pl.items || bytes == 0) return false;
  return k * dtype_size(x.dtype) <= 128 * bytes && pl.tile_rows * k <= kMaxEncoded && pl.channel_tiles * x.m * k * dtype_size(x.dtype) <= (16ll << 20);
}

template <typename T, typename O, int BYTES>
static cudaError_t launch(const CUtensorMap& map, const Params& p, unsigned grid, size_t smem, cudaStream_t st) {
  const bool two = (p.x.k1 + p.x.k2) * (int64_t)sizeof(T) <= 64 * BYTES;  // vectors a lane
  auto* kern = two ? linear_kernel<T, O, BYTES, 4, 2> : linear_kernel<T, O, BYTES, 2, 4>;
  if (allow_smem("int8_linear", (const void*)kern, kMaxSteps * kABytes + kMaxEncoded * 2 + 1024) != F2C_OK) return cudaErrorInvalidConfiguration;
  return launch_dependent(kern, dim3(grid), kThreads, smem, st, map, p);
}

template <typename T, typename O>
static cudaError_t by_width(const CUtensorMap& map, const Params& p, unsigned grid, size_t smem, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (width(p.x) == 8) return launch<T, O, 8>(map, p, grid, smem, st);
  }
  return launch<T, O, 16>(map, p, grid, smem, st);
}

template <typename T>
static cudaError_t by_output(int out_dtype, const CUtensorMap& map, const Params& p, unsigned grid, size_t smem, cudaStream_t st) {
  if (out_dtype == F2C_F32) return by_width<T, float>(map, p, grid, smem, st);
  if (out_dtype == F2C_F16) return by_width<T, __half>(map, p, grid, smem, st);
  return by_width<T, __nv_bfloat16>(map, p, grid, smem, st);
}

static int run(const char* op, const Rows& x, const Job& j, const Plan& pl, cudaStream_t st) {
  CUtensorMap map;
  F2C_REQUIRE(make_map(&map, j.b.p, 1, j.b.rows, j.k, j.b.ld, kM), F2C_ERR_CUDA, "%s: tensor map", op);
  const Params p{x, j.b_scales, j.bias, j.out, (int)j.b.rows, pl.steps, pl.channel_tiles, pl.tile_rows, pl.tmem, j.relu, j.tries, stream_error_word()};
  const size_t smem = (size_t)pl.steps * (kABytes + (size_t)pl.tile_rows * kK) + 1024;
  const cudaError_t e = x.dtype == F2C_F32   ? by_output<float>(j.out_dtype, map, p, pl.grid, smem, st)
                        : x.dtype == F2C_F16 ? by_output<__half>(j.out_dtype, map, p, pl.grid, smem, st)
                                             : by_output<__nv_bfloat16>(j.out_dtype, map, p, pl.grid, smem, st);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return set_error(F2C_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
  }
  return check_launch(op);
}

}  // namespace i8l
}  // namespace f2c

using namespace f2c;

extern "C" int64_t f2c_int8_linear_workspace(const void* x1, int64_t ld1, int64_t k1, const void* x2, int64_t ld2, int64_t k2, int dtype, const int8_t* w,
                                             int64_t ldw, int64_t m, int64_t n) {
  const int64_t k = k1 + k2, ld = i8::round16(k);
  if (m < 1 || n < 1 || k < 0 || k > i8::kMaxK) return 0;
  const i8::Rows r{x1, x2, ld1, ld2, k1, k2, m, dtype};  // (which way it goes hangs on their alignment)
  const int64_t rows = i8::few_encodes(r, n) || i8l::one_launch(r, i8::plan(m, n, k, current_sm_count())) ? 0 : i8::round256(4 * m) + i8::round256(m * ld);
  return rows + (k == 0 || i8::in_place(w, ldw, n) ? 0 : i8::round256(n * ld));
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
  const int64_t need = f2c_int8_linear_workspace(x1, ld1, k1, x2, ld2, k2, dtype, w, ldw, m, n);
  F2C_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), F2C_ERR_INVALID,
              "%s: workspace too small or not 256-byte aligned", op);
  cudaStream_t st = (cudaStream_t)stream;
  char* ws = (char*)workspace;
  i8::Job j{};
  j.a_scales = nullptr; j.b_scales = w_scales; j.bias = bias; j.out = out; j.k = k; j.out_dtype = out_dtype;
  j.activation(relu);
  if (i8::few_encodes(r, n)) {
    j.b = i8::readable(i8::Operand{w, ldw, n}, k, ws, st);
    return i8::few(op, r, j, st);
  }
  const i8::Plan pl = i8::plan(m, n, k, current_sm_count());
  if (i8l::one_launch(r, pl)) {
    j.b = i8::readable(i8::Operand{w, ldw, n}, k, ws, st);
    return i8l::run(op, r, j, pl, st);
  }
  float* scales = (float*)ws;
  ws += i8::round256(4 * m);
  int8_t* codes = (int8_t*)ws;
  const int64_t ldq = i8::round16(k);
  ws += i8::round256(m * ldq);
  j.b = i8::readable(i8::Operand{w, ldw, n}, k, ws, st);  // before the rows: the product may then ask for weights while these are encoded
  if (const int rc = i8::quantize(r, codes, ldq, scales, st)) return rc;
  j.a = i8::Operand{codes, ldq, m};
  j.a_scales = scales; j.weights_first = 1;
  return i8::mm(op, j, st);
}
