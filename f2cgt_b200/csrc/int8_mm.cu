// out [m, n] = act(s[i] ws[j] sum_t q[i, t] w[j, t] + b[j]) in 8-bit integers on the 5th-generation tensor cores (f2c_int8_mm,
// f2c_int8_linear).
//
// A tile of the product has 128 channels (rows of w, the lanes of TMEM) and up to 256 rows of q (its columns), whatever m: the weights are
// what few rows have to read, and they fill the MMA's 128 rows; an epilogue thread has one channel, whose scale and bias stay in
// registers, and a warp writes 32 neighbouring channels of a row of out without staging them.  128 columns of K come per step with TMA
// (128-byte swizzle, zeros behind the operands' edges) through a ring of stages; the int32 accumulators of two tiles alternate in TMEM.
//  * Rows per tile: so many that the SMs have equal work in few rounds (see plan()).
//  * Many tiles and a long K: pairs of CTAs share a tile of 256 channels, so that each fetches half of the rows: 32 KB for a step of K instead of 48.
//  * Few tiles and a long K: the CTAs of a cluster each take a part of K and add their sums over distributed shared memory, which is exact
//    and in any order the same.
// Large products are bound by the tensor cores (16,384 x 4096 x 4096: 166 us, 3.3 POP/s, the tensor pipe busy 94% of the time), those of short K by
// memory (59,000 x 128 x 256 to float32: 10.6 us a call, 4.3 TB/s), small ones by latency (16 x 4096 x 4096 with the codes of its rows: 7.3 us).
// Every wait is bounded: when one runs out the CTA's roles all leave, what it has not finished becomes NaN, copies and products in flight are
// waited for, the error word is raised and TMEM is freed.
#include "int8_mm.cuh"

#include <algorithm>
#include <climits>

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
  int stages, split, relu;
  int tmem, accumulators;   // columns of an accumulator, and how many
  int parts_at, share_log;  // clusters: where the sums are in shared memory, and of how many rows
  int weights_first;        // the kernel before this one does not make the weights
  uint32_t tries;           // of a role's bounded waits; 0: nothing is issued
  int* error;
};

struct Bars {
  uint64_t full[kMaxStages], empty[kMaxStages], drain, acc_full[2], acc_empty[2];
  uint32_t tmem;
  int failed, lost;  // lost: of any CTA of the cluster
};

// CTAS 2: the two CTAs of a cluster work on 256 channels, each with 128 of them and half of the tile's rows in its shared memory; the first one
// issues the MMAs for both.
template <typename T, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS == 1 ? 2 : 1) mm_kernel(const __grid_constant__ CUtensorMap codes, const __grid_constant__ CUtensorMap w, const Params p) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ Bars bars;
  __shared__ __align__(16) float scales_s[kEpilogueWarps][kMaxN];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  const int split = CTAS == 1 ? p.split : 1, group = split * CTAS;
  const int rank = (int)blockIdx.x % group, first = (int)blockIdx.x / group, stride = (int)gridDim.x / group;
  const int part = CTAS == 1 ? rank : 0;  // of K
  const int step0 = (int)((int64_t)p.steps * part / split), steps = (int)((int64_t)p.steps * (part + 1) / split) - step0;
  const int tile_channels = kM * CTAS, b_rows = p.tile_rows / CTAS, own_channels = CTAS == 1 ? 0 : rank * kM, own_rows = CTAS == 1 ? 0 : rank * b_rows;
  const uint32_t b_bytes = (uint32_t)b_rows * kK;
  const uint32_t stage_bytes = (uint32_t)kABytes + b_bytes;
  uint32_t left = p.tries;

  if (wid == 1) {
    if (CTAS == 2) alloc_tmem_pair(&bars.tmem, (uint32_t)p.tmem * p.accumulators);
    else alloc_tmem(&bars.tmem, (uint32_t)p.tmem * p.accumulators);
  }
  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) { init_bar(bars.full + s, 1); init_bar(bars.empty + s, 1); }
    init_bar(&bars.drain, 1);
    for (int b = 0; b < 2; ++b) { init_bar(bars.acc_full + b, 1); init_bar(bars.acc_empty + b, kEpilogueWarps * CTAS); }
    fence_bars();
    bars.failed = 0;
    bars.lost = 0;
  }
  fence_before();
  __syncthreads();
  if (group > 1) cluster_barrier();  // all are here before the first tells another its sums, or that it has loaded
  fence_after();
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
    const uint32_t ring = smem_u32(smem), bars0 = CTAS == 2 ? peer_address(smem_u32(bars.full), 0) : smem_u32(bars.full);
    const auto load = [&](bool go, const CUtensorMap* map, uint32_t dst, uint32_t bar, int x, int y) {
      if (CTAS == 2) tma_load_pair(go, map, dst, bar, x, y);
      else tma_load(go, map, dst, bar, x, y);
    };
    const bool counts = CTAS == 1 || rank == 0;  // the first one's barriers count the bytes of both
    int ahead = 0;  // stages whose weights have been asked for
    if (p.weights_first) {
      for (; ahead < min(p.stages, steps); ++ahead) {
        expect_if(mine && left != 0u && counts, bars.full + ahead, stage_bytes * CTAS);
        load(mine && left != 0u, &w, ring + (uint32_t)ahead * stage_bytes, bars0 + 8u * (uint32_t)ahead, (step0 + ahead) * kK, first % p.channel_tiles * tile_channels + own_channels);
      }
      dependency_wait();
    }
    release_dependents();
    for (int item = first; item < p.items; item += stride) {
      const int channel0 = item % p.channel_tiles * tile_channels + own_channels, row0 = item / p.channel_tiles * p.tile_rows + own_rows;
      for (int i = 0; i < steps; ++i) {
        if (round > 0) wait_bar(bars.empty + s, (round - 1) & 1, left);
        const bool go = mine && left != 0u, fresh = go && (round > 0 || s >= ahead);
        const uint32_t stage = ring + (uint32_t)s * stage_bytes, bar = bars0 + 8u * (uint32_t)s;
        expect_if(fresh && counts, bars.full + s, stage_bytes * CTAS);
        load(fresh, &w, stage, bar, (step0 + i) * kK, channel0);
        load(go, &codes, stage + (uint32_t)kABytes, bar, (step0 + i) * kK, row0);
        if (++s == p.stages) { s = 0; ++round; }
      }
    }
  } else if (wid == 1) {
    // ================= MMAs
    const bool mine = elected() != 0u;
    const uint32_t idesc = instruction(kSumS32, kFormatS8, kM * CTAS, (uint32_t)p.tile_rows);
    const uint32_t a_low = desc_low(smem_u32(smem), kChunkAlongK), b_low = a_low + (kABytes >> 4);
    const auto done = [&](bool go, const uint64_t* bar) {
      if (CTAS == 2) commit_pair(go, bar);
      else commit(go, bar);
    };
    uint32_t t = 0;
    for (int item = CTAS == 1 || rank == 0 ? first : p.items; item < p.items; item += stride, ++t) {
      const uint32_t buf = t & 1u, acc = tmem + buf * (uint32_t)p.tmem;
      if (t >= 2) wait_bar(bars.acc_empty + buf, ((t >> 1) - 1) & 1, left);
      for (int i = 0; i < steps; ++i) {
        wait_bar(bars.full + s, round & 1, left);
        fence_after();
        const bool go = mine && left != 0u;
        const uint32_t at = (uint32_t)s * (stage_bytes >> 4), a = a_low + at, b = b_low + at;
#pragma unroll
        for (uint32_t q = 0; q < kK / 32; ++q) {
          if (CTAS == 2) mma_i8_pair(go, acc, desc(a + q * kStepAlongK), desc(b + q * kStepAlongK), idesc, i + (int)q != 0);
          else mma_i8(go, acc, desc(a + q * kStepAlongK), desc(b + q * kStepAlongK), idesc, i + (int)q != 0);
        }
        done(go, bars.empty + s);
        if (++s == p.stages) { s = 0; ++round; }
      }
      done(mine && left != 0u, bars.acc_full + buf);
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
      const int channel = item % p.channel_tiles * tile_channels + own_channels + quarter * 32 + lane;
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
        if (split > 1) {
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
      if (split > 1 && lost && lane < split) peer_store(peer_address(smem_u32(&bars.lost), (uint32_t)lane), 1u);
      // the accumulators have been read
      fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CTAS == 2) peer_arrive(peer_address(smem_u32(bars.acc_empty + buf), 0));
        else arrive(bars.acc_empty + buf);
      }
    }
  }
  if (left == 0u) bars.failed = 1;
  if (split > 1) {
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
          if (q < split) sum += part[(q * share + i) * kM];
        if (mine) ((T*)p.out)[(row0 + c) * p.n + channel] = from_float<T>(finish(sum, scales_s[wid - 2][c] * w_scale, bias, floor));
      }
    }
  }
  fence_before();
  __syncthreads();
  if (bars.failed && p.tries != 0u && (CTAS == 1 || rank == 0)) {
    // copies in flight write to shared memory, MMAs in flight read it and write TMEM, of both CTAs of a pair: wait (bounded) for what was issued
    left = p.tries;
    if (wid == 0) {
      for (int q = 0; q < p.stages; ++q) {
        const uint32_t uses = round + (q < s ? 1u : 0u);
        if (uses > 0) wait_bar(bars.full + q, (uses - 1) & 1, left);
      }
    } else if (wid == 1) {
      const bool mine = elected() != 0u;  // who issued them
      if (CTAS == 2) commit_pair(mine, &bars.drain, 1);
      else commit(mine, &bars.drain);
      wait_bar(&bars.drain, 0, left);
    }
    __syncthreads();
  }
  if (CTAS == 2) cluster_barrier();
  if (wid == 1) {
    fence_after();
    if (CTAS == 2) free_tmem_pair(tmem, (uint32_t)p.tmem * p.accumulators);
    else free_tmem(tmem, (uint32_t)p.tmem * p.accumulators);
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
  const int channel_tiles = (int)ceil_div(n, kM);
  p.steps = (int)ceil_div(k, kK);
  // Rows per tile, CTAs that share them and parts of K: the choice of least cycles.
  const size_t room = kRoom - 1024;
  int64_t least = INT64_MAX;
  const auto consider = [&](int rows, int ctas, int split) {
    Plan q{};
    q.steps = p.steps;
    q.tile_rows = rows;
    q.ctas = ctas;
    q.split = split;
    q.channel_tiles = (channel_tiles + ctas - 1) / ctas;
    q.items = (int)(ceil_div(m, rows) * q.channel_tiles);
    const int most = sms / (ctas * split);  // at a time
    const int at_once = q.items < most ? q.items : most;
    const size_t b_bytes = (size_t)rows / ctas * kK, parts = split > 1 ? (size_t)rows * kM * 4 : 0;
    q.grid = (unsigned)(at_once * ctas * split);
    const size_t stage = kABytes + b_bytes;
    const int steps = (q.steps + split - 1) / split, rounds = (q.items + at_once - 1) / at_once;
    q.accumulators = rounds > 1 ? 2 : 1;
    q.stages = (int)((room - parts) / stage);
    if (q.stages > kMaxStages) q.stages = kMaxStages;
    // A step of K takes the longest of its bytes at 56 a cycle (what an SM was seen to get from L2 with all others at it; 100 where half of them
    // have none), its MMAs, and the 2800 cycles that memory was seen to take under load shared among the stages; the results 12 cycles a row,
    // beside the next tile's steps; a tile 1000; the exchange between the parts of K 2000 and 16 a row; a pair 100 a step and 1500.  What it chooses between, measured
    // (calls in a graph, to bfloat16 but for *, which is to float32; inputs and results that L2 does not hold):
    //   16384 x 4096 x 4096 (m x n x k): 192 us with 256 rows and a CTA, 164 with a pair; 30000 x 400 x 3000: 46, 39, and 37 with 224 rows and a pair
    //   512 x 4096 x 4096: 11.3 us with 128 rows and a CTA, 10.7 with a pair, 13.2 with 192 rows, 13.8 with 64
    //   59,000 x 128 x 256 *: 11.8 us with 224 rows, 11.9 with 256, 13.0 with 128; 20,000 x 128 x 256 *: 6.0 with 160, 6.2 with 192, 7.7 with 128
    //   32 x 4096 x 4096: 7.5 us in four parts of K, 7.9 in two, 8.0 in one; 128 x 4096 x 4096 (64 rows): 8.5 in one, 10.0 in two
    // (Weights kept in shared memory over a CTA's tiles made no difference of 2% anywhere.)
    const int rate = 2 * (int)q.grid > sms ? 56 : 100, step = std::max(std::max((int)stage / rate + (ctas > 1 ? 100 : 0), 2 * rows), 2800 / q.stages);
    const int64_t tile = std::max((int64_t)steps * step, (int64_t)12 * rows);
    const int64_t cycles = rounds * (tile + 1000) + 12 * rows + (split > 1 ? 2000 + 16 * rows : 0) + (ctas > 1 ? 1500 : 0);
    if (cycles >= least) return;
    least = cycles;
    if ((int64_t)q.stages > (int64_t)rounds * steps) q.stages = rounds * steps > 0 ? rounds * steps : 1;
    q.tmem = 32;
    while (q.tmem < rows) q.tmem *= 2;
    q.parts_at = (int)(q.stages * stage);
    while ((split << q.share_log) < rows) ++q.share_log;
    q.smem = parts + q.stages * stage + 1024;
    p = q;
  };
  const bool fine = ceil_div(m, 64) * channel_tiles > sms;
  for (int rows = m > 16 ? 32 : 16; rows <= kMaxN; rows += fine && rows >= 64 ? 32 : rows) {  // (16 rows: as many steps for the weights as 32)
    const int64_t items = ceil_div(m, rows) * channel_tiles;
    const bool power = (rows & (rows - 1)) == 0;
    consider(rows, 1, 1);
    // (clusters do not fill the machine: 128 CTAs in clusters of 8, or 140 in clusters of 4, ran in two rounds)
    for (int split = 2; split <= kMaxSplit && power && items * split <= sms * (split < 8 ? 7 : 6) / 8 && p.steps >= 2 * split; split *= 2) consider(rows, 1, split);
    if (rows >= 64 && channel_tiles > 1) consider(rows, 2, 1);
    if (rows >= m) break;
  }
  return p;
}

template <int CTAS>
auto mm_kernel_of(int dtype) { return dtype == F2C_F32 ? mm_kernel<float, CTAS> : dtype == F2C_F16 ? mm_kernel<__half, CTAS> : mm_kernel<__nv_bfloat16, CTAS>; }

int mm(const char* op, const Job& j, cudaStream_t st) {
  const Plan pl = plan(j.a.rows, j.b.rows, j.k, current_sm_count());
  CUtensorMap maps[2] = {};
  if (j.k > 0) {
    const bool ok = make_map(maps, j.a.p, 1, j.a.rows, j.k, j.a.ld, pl.tile_rows / pl.ctas) && make_map(maps + 1, j.b.p, 1, j.b.rows, j.k, j.b.ld, kM);
    F2C_REQUIRE(ok, F2C_ERR_CUDA, "%s: tensor map", op);
  }
  Params p{j.a_scales, j.b_scales, j.bias, j.out, j.a.rows, (int)j.b.rows, pl.steps, pl.channel_tiles, pl.tile_rows, pl.items,
           pl.stages, pl.split, j.relu, pl.tmem, pl.accumulators, pl.parts_at, pl.share_log, j.weights_first, j.tries, stream_error_word()};
  auto* kern = pl.ctas == 2 ? mm_kernel_of<2>(j.out_dtype) : mm_kernel_of<1>(j.out_dtype);
  if (const int rc = allow_smem(op, (const void*)kern, (int)kRoom)) return rc;
  launch_dependent_cluster(kern, dim3(pl.grid), kThreads, pl.smem, (unsigned)(pl.split * pl.ctas), st, maps[0], maps[1], p);
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
  j.a_scales = scales; j.b_scales = w_scales; j.bias = bias; j.out = out; j.k = k; j.out_dtype = out_dtype;
  j.activation(relu);
  if (i8::is_few(m, n, k)) return i8::few(op, i8::Rows{j.a.p, nullptr, j.a.ld, 0, k, 0, m, F2C_I8}, j, st);
  return i8::mm(op, j, st);
}
