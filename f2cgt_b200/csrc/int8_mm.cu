// out [m, n] = act(s[i] ws[j] sum_t q[i, t] w[j, t] + b[j]) in 8-bit integers on the 5th-generation tensor cores (f2c_int8_mm,
// f2c_int8_linear).
//
// A tile of the product has 128 channels (rows of w, the lanes of TMEM) and up to 256 rows of q (its columns), whatever m: the weights are
// what few rows have to read, and they fill the MMA's 128 rows; an epilogue thread has one channel, whose scale and bias stay in
// registers, and a warp writes 32 neighbouring channels of a row of out without staging them.  128 columns of K come per step with TMA
// (128-byte swizzle, zeros behind the operands' edges) through a ring of stages; the int32 accumulators of two tiles alternate in TMEM.
//  * Rows per tile: so many that the tiles of one round over the SMs have equal work (see plan()).
//  * Short K and few channel tiles: a CTA keeps its channels' weights in shared memory and only the rows travel.
//  * Few tiles and a long K: the CTAs of a cluster each take a part of K and add their sums over distributed shared memory, which is exact
//    and in any order the same.
// Every wait is bounded: when one runs out the CTA's roles all leave, what it has not finished becomes NaN, copies and products in flight are
// waited for, the error word is raised and TMEM is freed.
#include "int8_mm.cuh"

namespace f2c {
namespace i8 {

constexpr int kEpilogueWarps = 8, kThreads = 64 + 32 * kEpilogueWarps;  // warp 0: TMA, warp 1: MMA, then the epilogue's
constexpr int kMaxStages = 12, kMaxSplit = 8;
constexpr size_t kRoom = kSmemLimit - 10240;  // dynamic shared memory: what barriers and scales leave, less the alignment of its start

struct Params {
  const float *a_scales, *b_scales, *bias;
  void* out;
  int64_t m;
  int n, steps;             // steps of K
  int channel_tiles, tile_rows, items;
  int stages, resident, split, relu;
  int tmem, accumulators;   // columns of an accumulator, and how many
  int parts_at, share_log;  // clusters: where the sums are in shared memory, and of how many rows
  int weights_first;        // the kernel before this one does not make the weights
  int* error;
};

struct Bars {
  uint64_t full[kMaxStages], empty[kMaxStages], weights, drain, acc_full[2], acc_empty[2];
  uint32_t tmem;
  int failed, lost;  // lost: of any CTA of the cluster
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) mm_kernel(const __grid_constant__ CUtensorMap codes, const __grid_constant__ CUtensorMap w, const Params p) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ Bars bars;
  __shared__ __align__(16) float scales_s[kEpilogueWarps][kMaxN];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  const int rank = (int)blockIdx.x % p.split, first = (int)blockIdx.x / p.split, stride = (int)gridDim.x / p.split;
  const int step0 = (int)((int64_t)p.steps * rank / p.split), steps = (int)((int64_t)p.steps * (rank + 1) / p.split) - step0;
  const uint32_t b_bytes = (uint32_t)p.tile_rows * kK;
  unsigned char* ring = smem + (p.resident ? (size_t)steps * kABytes : 0);
  const uint32_t stage_bytes = b_bytes + (p.resident ? 0u : (uint32_t)kABytes);
  uint32_t left = kWaitLimit;

  if (wid == 1) alloc_tmem(&bars.tmem, (uint32_t)p.tmem * p.accumulators);
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) { init_bar(bars.full + s, 1); init_bar(bars.empty + s, 1); }
    init_bar(&bars.weights, 1);
    init_bar(&bars.drain, 1);
    for (int b = 0; b < 2; ++b) { init_bar(bars.acc_full + b, 1); init_bar(bars.acc_empty + b, kEpilogueWarps); }
    fence_bars();
    bars.failed = 0;
    bars.lost = 0;
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (p.split > 1) cluster_barrier();  // all are here before the first tells another its sums
  const uint32_t tmem = bars.tmem;
  const int share = 1 << p.share_log;  // rows whose sums a CTA of a cluster adds up
  const uint32_t parts = smem_u32(smem) + (uint32_t)p.parts_at;
  int s = 0;
  uint32_t round = 0;

  if (wid == 0) {
    // ================= loads
    const bool mine = elected() != 0u;
    if (mine) {
      prefetch_map(&codes);
      prefetch_map(&w);
    }
    __syncwarp();
    if (!p.weights_first) dependency_wait();
    const uint32_t ring0 = smem_u32(ring), codes_at = p.resident ? 0u : (uint32_t)kABytes, bars0 = smem_u32(bars.full);
    int ahead = 0;  // stages whose weights have been asked for
    if (p.resident) {
      expect_if(mine, &bars.weights, (uint32_t)steps * kABytes);
      for (int i = 0; i < steps; ++i) tma_load(mine, &w, smem_u32(smem) + (uint32_t)i * kABytes, smem_u32(&bars.weights), (step0 + i) * kK, first % p.channel_tiles * kM);
    } else if (p.weights_first) {
      for (; ahead < min(p.stages, steps); ++ahead) {
        expect_if(mine, bars.full + ahead, stage_bytes);
        tma_load(mine, &w, ring0 + (uint32_t)ahead * stage_bytes, bars0 + 8u * (uint32_t)ahead, (step0 + ahead) * kK, first % p.channel_tiles * kM);
      }
    }
    if (p.weights_first) dependency_wait();
    release_dependents();
    for (int item = first; item < p.items; item += stride) {
      const int channel0 = item % p.channel_tiles * kM, row0 = item / p.channel_tiles * p.tile_rows;
      for (int i = 0; i < steps; ++i) {
        if (round > 0) wait_bar(bars.empty + s, (round - 1) & 1, left);
        const bool go = mine && left != 0u, fresh = go && (round > 0 || s >= ahead);
        const uint32_t stage = ring0 + (uint32_t)s * stage_bytes, bar = bars0 + 8u * (uint32_t)s;
        expect_if(fresh, bars.full + s, stage_bytes);
        tma_load(fresh && !p.resident, &w, stage, bar, (step0 + i) * kK, channel0);
        tma_load(go, &codes, stage + codes_at, bar, (step0 + i) * kK, row0);
        if (++s == p.stages) { s = 0; ++round; }
      }
    }
  } else if (wid == 1) {
    // ================= MMAs
    const bool mine = elected() != 0u;
    const uint32_t idesc = instruction(kSumS32, kFormatS8, kM, (uint32_t)p.tile_rows);
    const uint32_t a_low = desc_low(smem_u32(p.resident ? smem : ring), kChunkAlongK), b_low = desc_low(smem_u32(ring) + (p.resident ? 0 : kABytes), kChunkAlongK);
    if (p.resident) wait_bar(&bars.weights, 0, left);
    uint32_t t = 0;
    for (int item = first; item < p.items; item += stride, ++t) {
      const uint32_t buf = t & 1u, acc = tmem + buf * (uint32_t)p.tmem;
      if (t >= 2) wait_bar(bars.acc_empty + buf, ((t >> 1) - 1) & 1, left);
      for (int i = 0; i < steps; ++i) {
        wait_bar(bars.full + s, round & 1, left);
        fence_after();
        const bool go = mine && left != 0u;
        const uint32_t at = (uint32_t)s * (stage_bytes >> 4), a = a_low + (p.resident ? (uint32_t)i * (kABytes >> 4) : at), b = b_low + at;
#pragma unroll
        for (uint32_t q = 0; q < kK / 32; ++q) mma_i8(go, acc, desc(a + q * kStepAlongK), desc(b + q * kStepAlongK), idesc, i + (int)q != 0);
        commit(go, bars.empty + s);
        if (++s == p.stages) { s = 0; ++round; }
      }
      commit(mine && left != 0u, bars.acc_full + buf);
    }
  } else {
    // ================= epilogue: a warp has the TMEM lanes of its quarter and every other 32 rows of the tile, thread = channel
    const int quarter = wid & 3, half = (wid - 2) >> 2;
    float* row_scale = scales_s[wid - 2];
    const float floor = p.relu ? 0.0f : __int_as_float(0xff800000);
    uint32_t t = 0;
    dependency_wait();
    for (int item = first; item < p.items; item += stride, ++t) {
      const uint32_t buf = t & 1u;
      const int channel = item % p.channel_tiles * kM + quarter * 32 + lane;
      const int64_t row0 = (int64_t)(item / p.channel_tiles) * p.tile_rows;
      const int rows = (int)min((int64_t)p.tile_rows, p.m - row0);
      const bool mine = channel < p.n;
      const float w_scale = mine ? __ldg(p.b_scales + channel) : 0.0f, bias = mine && p.bias != nullptr ? __ldg(p.bias + channel) : 0.0f;
      for (int c = lane; c < rows; c += 32) row_scale[c] = __ldg(p.a_scales + row0 + c);
      __syncwarp();
      if (steps > 0) wait_bar(bars.acc_full + buf, (t >> 1) & 1, left);
      const bool lost = __any_sync(0xffffffffu, left == 0u);
      fence_after();
      const uint32_t at = tmem + ((uint32_t)(quarter * 32) << 16) + buf * (uint32_t)p.tmem;
      for (int c0 = half * 32; c0 < rows; c0 += 64) {
        uint32_t r[32];
        if (steps > 0) {
          tmem_ld32(at + (uint32_t)c0, r);
          tmem_wait(r);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = 0u;
        }
        if (p.split > 1) {
          // row c goes to CTA c / share, there [this CTA][c % share][channel]
          const uint32_t to = parts + 4u * (uint32_t)(rank * share * kM + quarter * 32 + lane);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c0 + j < rows) peer_store(peer_address(to + (uint32_t)((c0 + j) & (share - 1)) * (4u * kM), (uint32_t)(c0 + j) >> p.share_log), r[j]);
        } else if (mine) {
          store_rows((T*)p.out + (row0 + c0) * p.n + channel, (int64_t)p.n, r, row_scale + c0, w_scale, lost ? __int_as_float(0x7fffffff) : bias, floor, rows - c0);
        }
        __syncwarp();
      }
      if (p.split > 1 && lost && lane < p.split) peer_store(peer_address(smem_u32(&bars.lost), (uint32_t)lane), 1u);
      // the accumulators have been read
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(bars.acc_empty + buf);
    }
  }
  if (left == 0u) bars.failed = 1;
  if (p.split > 1) {
    // a cluster has one tile, whose rows its CTAs share: all sums have been told when all have got here
    __syncwarp();
    cluster_barrier();
    if (wid >= 2) {
      const int quarter = wid & 3, half = (wid - 2) >> 2, channel = first % p.channel_tiles * kM + quarter * 32 + lane;
      const int64_t row0 = (int64_t)(first / p.channel_tiles) * p.tile_rows;
      const int rows = (int)min((int64_t)p.tile_rows, p.m - row0);
      const bool mine = channel < p.n;
      const float w_scale = mine ? __ldg(p.b_scales + channel) : 0.0f;
      const float bias = bars.lost ? __int_as_float(0x7fffffff) : mine && p.bias != nullptr ? __ldg(p.bias + channel) : 0.0f;
      const float floor = p.relu ? 0.0f : __int_as_float(0xff800000);
      const int* part = reinterpret_cast<const int*>(smem + p.parts_at) + quarter * 32 + lane;
#pragma unroll 2
      for (int i = half; i < share; i += 2) {
        const int c = rank * share + i;
        if (c >= rows) break;
        int sum = 0;
#pragma unroll
        for (int q = 0; q < kMaxSplit; ++q)
          if (q < p.split) sum += part[(q * share + i) * kM];
        if (mine) ((T*)p.out)[(row0 + c) * p.n + channel] = from_float<T>(finish(sum, scales_s[wid - 2][c] * w_scale, bias, floor));
      }
    }
  }
  fence_before();
  __syncthreads();
  if (bars.failed) {
    // copies in flight write to this CTA's shared memory, MMAs in flight read it and write its TMEM: wait (bounded) for what was issued
    left = kWaitLimit;
    if (tid == 0) {
      if (p.resident) wait_bar(&bars.weights, 0, left);
      for (int q = 0; q < p.stages; ++q) {
        const uint32_t uses = round + (q < s ? 1u : 0u);
        if (uses > 0) wait_bar(bars.full + q, (uses - 1) & 1, left);
      }
    } else if (tid == 32) {
      commit(true, &bars.drain);
      wait_bar(&bars.drain, 0, left);
    }
    __syncthreads();
  }
  if (wid == 1) {
    fence_after();
    free_tmem(tmem, (uint32_t)p.tmem * p.accumulators);
  }
  if (tid == 0 && bars.failed) report_wait(p.error, 4);
}

// Copies codes to rows that start on 16 bytes.
__global__ void __launch_bounds__(256) align_kernel(const int8_t* __restrict__ src, int64_t ld, int64_t k, int8_t* __restrict__ dst, int64_t aligned_ld, int64_t rows) {
  dependency_wait();
  release_dependents();
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
    for (int64_t t = threadIdx.x; t < k; t += 256) dst[row * aligned_ld + t] = src[row * ld + t];
}

// The operand where TMA can read it: its own memory, or a copy in the workspace (which moves on).
Operand readable(const Operand& o, int64_t k, char*& ws, cudaStream_t st) {
  const int64_t ld = round16(k);
  if (k == 0 || in_place(o.p, o.ld, o.rows)) return Operand{o.p, o.rows > 1 ? o.ld : ld, o.rows};
  int8_t* copy = (int8_t*)ws;
  ws += round256(o.rows * ld);
  launch_dependent(align_kernel, dim3((unsigned)(o.rows < 4096 ? o.rows : 4096)), 256, 0, st, o.p, o.ld, k, copy, ld, o.rows);
  return Operand{copy, ld, o.rows};
}

static_assert(sizeof(Bars) + kEpilogueWarps * kMaxN * 4 + 256 <= 10240, "static shared memory");

int check(const char* op, int64_t m, int64_t n, int64_t k, int out_dtype) {
  F2C_REQUIRE(m >= 0 && n >= 0 && k >= 0, F2C_ERR_INVALID, "%s: negative size", op);
  F2C_REQUIRE(is_float_dtype(out_dtype), F2C_ERR_UNSUPPORTED, "%s: the output must be float32, float16 or bfloat16", op);
  F2C_REQUIRE(k <= kMaxK, F2C_ERR_LIMIT, "%s: more than %d columns", op, kMaxK);
  F2C_REQUIRE(m <= kMaxRows && n <= (1 << 21), F2C_ERR_LIMIT, "%s: too many rows", op);
  return F2C_OK;
}

Plan plan(int64_t m, int64_t n, int64_t k, int sms) {
  Plan p{};
  p.channel_tiles = (int)ceil_div(n, kM);
  p.steps = (int)ceil_div(k, kK);
  // Rows per tile and parts of K: the pair of least cycles.  A step of K takes the longer of its bytes at 56 a cycle (what an SM was seen
  // to get from L2 with all others at it) and its MMAs; the results 12 cycles a row, beside the next tile's steps; a tile 1000 more;
  // the exchange between the parts of K 2000 and 16 a row.  (59,000 x 128 x 256: 9.2 us with 256 rows, 10.0 with 96, 11.6 with 64; 2000 x 1000 x 500:
  // 5.5 us with 128, 6.5 with 64, 6.4 with 256.)
  const size_t room = kRoom - 1024, weights = (size_t)p.steps * kABytes;
  int64_t least = 0;
  for (const int rows : {16, 32, 64, 128, 192, 256}) {
    if (rows == 16 && m > 16) continue;  // as many steps for the weights as 32
    const int64_t items = ceil_div(m, rows) * p.channel_tiles;
    for (int split = 1; split <= kMaxSplit; split *= 2) {
      if (split > 1 && (items * split > sms || p.steps < 2 * split || rows == 192)) break;
      const int64_t rounds = ceil_div(items * split, sms), steps = ceil_div(p.steps, split);
      const bool resident = split == 1 && sms >= p.channel_tiles && weights + 4 * rows * kK <= room;
      const int64_t bytes = rows * kK + (resident ? 0 : kABytes), step = bytes / 56 > 2 * rows ? bytes / 56 : 2 * rows;
      const int64_t tile = steps * step > 12 * rows ? steps * step : 12 * rows;
      const int64_t cycles = rounds * (tile + 1000) + 12 * rows + (resident ? (int64_t)weights / 56 : 0) + (split > 1 ? 2000 + 16 * rows : 0);
      if (least != 0 && cycles >= least) continue;
      least = cycles;
      p.tile_rows = rows;
      p.split = split;
    }
    if (rows >= m) break;
  }
  const int64_t items = ceil_div(m, p.tile_rows) * p.channel_tiles;
  p.items = (int)items;
  const size_t b_bytes = (size_t)p.tile_rows * kK;
  int64_t clusters = items;
  if (p.split == 1 && items > sms) clusters = sms;
  if (p.split == 1 && sms >= p.channel_tiles && weights + 4 * b_bytes <= room) {
    p.resident = 1;
    const int64_t whole = (int64_t)sms / p.channel_tiles * p.channel_tiles;  // a CTA stays with its channels
    if (clusters > whole) clusters = whole;
  }
  p.grid = (unsigned)(clusters * p.split);
  p.tmem = 32;
  while (p.tmem < p.tile_rows) p.tmem *= 2;
  const size_t parts = p.split > 1 ? (size_t)p.tile_rows * kM * 4 : 0;
  const size_t stage = b_bytes + (p.resident ? 0 : kABytes), fixed = (p.resident ? weights : 0) + parts;
  const int64_t most = p.rounds() * ceil_div(p.steps, p.split);
  p.stages = (int)((room - fixed) / stage);
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  if (p.stages > most) p.stages = (int)(most > 0 ? most : 1);
  p.parts_at = (int)(p.stages * stage);  // (never resident)
  while ((p.split << p.share_log) < p.tile_rows) ++p.share_log;
  p.smem = fixed + p.stages * stage + 1024;
  return p;
}

int mm(const char* op, const Job& j, cudaStream_t st) {
  const Plan pl = plan(j.a.rows, j.b.rows, j.k, current_sm_count());
  CUtensorMap maps[2] = {};
  if (j.k > 0) {
    const bool ok = make_map(maps, j.a.p, 1, j.a.rows, j.k, j.a.ld, pl.tile_rows) && make_map(maps + 1, j.b.p, 1, j.b.rows, j.k, j.b.ld, kM);
    F2C_REQUIRE(ok, F2C_ERR_CUDA, "%s: tensor map", op);
  }
  Params p{j.a_scales, j.b_scales, j.bias, j.out, j.a.rows, (int)j.b.rows, pl.steps, pl.channel_tiles, pl.tile_rows, pl.items,
           pl.stages, pl.resident, pl.split, j.relu, pl.tmem, pl.rounds() > 1 ? 2 : 1, pl.parts_at, pl.share_log, j.weights_first, stream_error_word()};
  auto* kern = j.out_dtype == F2C_F32 ? mm_kernel<float> : j.out_dtype == F2C_F16 ? mm_kernel<__half> : mm_kernel<__nv_bfloat16>;
  if (const int rc = allow_smem(op, (const void*)kern, (int)kRoom)) return rc;
  launch_dependent_cluster(kern, dim3(pl.grid), kThreads, pl.smem, (unsigned)pl.split, st, maps[0], maps[1], p);
  return check_launch(op);
}

}  // namespace i8
}  // namespace f2c

using namespace f2c;

extern "C" int64_t f2c_int8_mm_workspace(const int8_t* codes, int64_t ldq, const int8_t* w, int64_t ldw, int64_t m, int64_t n, int64_t k) {
  if (m < 1 || n < 1 || k < 1) return 0;
  const int64_t ld = i8::round16(k);
  return (i8::in_place(codes, ldq, m) ? 0 : i8::round256(m * ld)) + (i8::in_place(w, ldw, n) ? 0 : i8::round256(n * ld));
}

extern "C" int f2c_int8_mm(const int8_t* codes, int64_t ldq, const float* scales, const int8_t* w, int64_t ldw, const float* w_scales,
                           const float* bias, int relu, void* out, int out_dtype, int64_t m, int64_t n, int64_t k, void* workspace,
                           int64_t workspace_bytes, void* stream) {
  const char* op = "int8_mm";
  if (const int rc = i8::check(op, m, n, k, out_dtype)) return rc;
  F2C_REQUIRE((m <= 1 || ldq >= k) && (n <= 1 || ldw >= k), F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  if (m == 0 || n == 0) return F2C_OK;
  F2C_REQUIRE(out && scales && w_scales && (k == 0 || (codes && w)), F2C_ERR_INVALID, "%s: null pointer", op);
  const int64_t need = f2c_int8_mm_workspace(codes, ldq, w, ldw, m, n, k);
  F2C_REQUIRE(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), F2C_ERR_INVALID,
              "%s: workspace too small or not 256-byte aligned", op);
  cudaStream_t st = (cudaStream_t)stream;
  char* ws = (char*)workspace;
  i8::Job j{};
  j.a = i8::readable(i8::Operand{codes, ldq, m}, k, ws, st);
  j.b = i8::readable(i8::Operand{w, ldw, n}, k, ws, st);
  j.a_scales = scales; j.b_scales = w_scales; j.bias = bias; j.out = out; j.k = k; j.relu = relu; j.out_dtype = out_dtype;
  if (i8::is_few(m, n, k)) return i8::few(op, i8::Rows{j.a.p, nullptr, j.a.ld, 0, k, 0, m, F2C_I8}, j, st);
  return i8::mm(op, j, st);
}
