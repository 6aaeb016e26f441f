// Gradient of a linear layer's weight and bias, its input kept in 8 bits (f2c_checkpoint_weight_grad):
//   dW[i, j] = sum over rows r of dy[r, i] x[r, j],  x[r, j] = low[r, g] + step[r, g] q[r, j],  g the group of column j;  db[i] = sum over rows of dy[r, i],
// on the 5th-generation tensor cores.  The input is never written out: it is decoded between shared memory and the tensor cores.  32 rows of dy and of codes
// at a time come with TMA through a ring of stages; four groups of four warps take the stages in turn, a thread has a column; one operand goes to TMEM by
// way of their registers, the other one lies in shared memory along M or N, which the MMA takes as it is.
//
//  * bfloat16 dy (rows_kernel).  dy is an operand as it is.  x is two bfloat16 numbers, 16 bits, of a product that is rounded to 8: two MMAs of
//    128 columns of x (the lanes of TMEM) by 256 of dy for every 16 rows.
//  * float32 and float16 dy (scaled_kernel).  With the factors taken to the other side, dW = (step dy)^T (q - z) + (base dy)^T 1, base = low + step z: differences of
//    codes, -255 .. 255, are bfloat16 numbers as they are, and step dy, rounded to single precision, is a sum of three of them (its 24 bits, eight each; float32) or two
//    (16 bits; float16, whose range bfloat16 has and float16 values of x might leave).  The second term is one number for every column of dy and group, summed in
//    registers.  z is the code nearest to a value of zero: then no |base| is more than |x|, and no step |q - z| more than 2 |x|, so that neither sum is large where the result is
//    not.  (With z = 0 both had the size of the groups' ranges and cancelled, and a small value beside large ones lost most of its digits; 16,384 x 1700 x 1700 float32
//    358 us so and 368 with z.)  128 columns of dy (the lanes) by a group.
//
// Sums.  The tensor cores cut sums off instead of rounding them, for every 16 rows and all one way: 16,384 rows of bfloat16 lost 4e-5 of their sums, and so 4e-4 of
// the norm of the rounded results.  So they are taken out and added up in single precision, every 256 rows (float32) or 1024 (float16; 16,384 x 1700 x 1700 401 us, and
// 395 every 16,384) in registers, while the MMAs go on in the other half of the accumulators; for bfloat16, whose accumulators leave no room for a second half, every
// 2048 rows, in shared memory and TMEM, while the MMAs wait (16,384 x 2048 x 4096, side by side: 488 us without, 495 every 4096 rows, 507 every 2048, 533 every 1024).
//
// What bounds it: bfloat16 shared memory, from which a stage's operand is read twice while its codes and steps are read and the next stages arrive (16,384 x 2048 x
// 4096: 515 us among other calls, 534 TFLOP/s of the product, 1070 of the MMAs, 480 by itself; half the MMAs, or no reading of codes and steps, each took 20% off); float32 the instructions that
// split dy times the step, 650 a warp for a stage (4096 x 2048 x 1152: 74 us); few rows latency (59,000 x 128 x 128 float32: 17 us of 5.9 that memory takes).
//
// Many rows and few tiles: the rows are dealt out over all SMs; each leaves its part of the sums, and a second launch adds them up in their order.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "checkpoint.cuh"
#include "tcgen05.cuh"

namespace f2c {
namespace wg {

using namespace t5;
using ckpt::both;
using ckpt::f32x2;
using ckpt::fma2;
using ckpt::kGroup;
using ckpt::mul2;
using ckpt::pair_of;
using ckpt::plus2;

constexpr int kGroups = 4, kWarps = 4 * kGroups, kThreads = 32 * (kWarps + 2);  // then a warp for the loads and one for the MMAs
constexpr int kRows = 32, kStages = 8;
constexpr uint32_t kBox = kRows * 128;  // a stage's rows of 128 bytes
constexpr uint32_t kFormatBf16 = 1;
constexpr int64_t kMaxSplitRows = 65536;

struct Params {
  const float* scales;
  int64_t groups, m;
  int n, k;
  int n_tiles, splits;
  int whole, rest;        // tiles that one CTA has all rows of, and the others, whose rows are split
  int64_t split_rows;     // a multiple of kRows
  void *dw, *db;          // of dy's type
  float *part, *part_db;  // (splits > 1) [split][tile of the others][columns / 4][128][4], and (nothing whole) [split][n_tiles * columns of dy]
  uint32_t tries;
  int* error;
};

struct Bars {
  uint64_t full[kStages], empty[kStages], ready[kGroups], taken[kGroups], drain, acc_full[2], acc_empty[2];
  uint32_t tmem;
  int failed;
};

// The MMA whose first operand is in TMEM, two 16-bit elements of K to a column.
__device__ __forceinline__ void mma_f16_tmem(bool go, uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, g;\n\tsetp.ne.b32 g, %6, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@g tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d_tmem), "r"(a_tmem), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(0u),
      "r"((uint32_t)go)
      : "memory");
}
// 32, 16 or 8 columns of the 32 lanes that the warp owns
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
      "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t pack_bf16(f32x2 v) {  // round to even
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi32(v)), "f"(lo32(v)));
  return r;
}
// the same cut off
__device__ __forceinline__ uint32_t cut_bf16(f32x2 v) { return __byte_perm((uint32_t)v, (uint32_t)(v >> 32), 0x7632); }
// v less the two numbers of w: exact where they are v rounded or cut off
__device__ __forceinline__ f32x2 less_bf16(f32x2 v, uint32_t w) { return fma2(pair_of(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)), both(-1.0f), v); }
__device__ __forceinline__ uint32_t lds_u8(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t at) {
  uint32_t v;
  asm volatile("{\n\t.reg .u16 h;\n\tld.shared.u16 h, [%1];\n\tcvt.u32.u16 %0, h;\n\t}" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds_u32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint4 lds_u128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ void sts_u128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// The steps and lowest values of a stage's rows, for a warp: lane r has row r's on the way a round ahead, and all get them from shared memory.
struct Scales {
  uint2 next;
  __device__ __forceinline__ void fetch(const Params& p, int64_t row0, int64_t rows, int stage, int group) {
    const int64_t r = (int64_t)stage * kRows + (threadIdx.x & 31);
    next = ldg_nc_u64_if(p.scales + 2 * ((row0 + r) * p.groups + group), r < rows);
  }
  // [steps of 32 rows][lowest values]
  __device__ __forceinline__ void tell(float* mine) const {
    const int lane = threadIdx.x & 31;
    __syncwarp();  // (the ones before have been read)
    mine[lane] = __uint_as_float(next.x);
    mine[32 + lane] = __uint_as_float(next.y);
    __syncwarp();
  }
  // [steps of 32 rows][values of the codes z nearest to zero][2^23 + z]
  __device__ __forceinline__ void tell_about_zero(float* mine) const {
    const int lane = threadIdx.x & 31;
    const float step = __uint_as_float(next.x), low = __uint_as_float(next.y);
    const float z = fminf(fmaxf(rintf(__fdividef(-low, step)), 0.0f), 255.0f);  // (any code is right; 0 where there is no quotient)
    __syncwarp();
    mine[lane] = step;
    mine[32 + lane] = fmaf(step, z, low);
    mine[64 + lane] = 8388608.0f + z;
    __syncwarp();
  }
};

struct Place {
  int split, n0, group;
  int part;  // -1: the result itself
  int64_t row0, rows;
  int stages;
  __device__ __forceinline__ Place(const Params& p, int columns) {
    const int other = (int)blockIdx.x - p.whole, tile = other < 0 ? (int)blockIdx.x : p.whole + other / p.splits;
    split = other < 0 ? 0 : other % p.splits;
    part = other < 0 || p.splits == 1 ? -1 : split * p.rest + (tile - p.whole);
    n0 = tile % p.n_tiles * columns;
    group = tile / p.n_tiles;
    row0 = split * p.split_rows;
    rows = other < 0 ? p.m : min(p.split_rows, p.m - row0);
    stages = (int)((rows + kRows - 1) / kRows);
  }
};

// Barriers and TMEM (512 columns: no other CTA that has any is on the SM, which the shared memory sees to)
__device__ __forceinline__ void begin(Bars& bars, uint32_t empties) {
  if (threadIdx.x / 32 == kWarps + 1) alloc_tmem(&bars.tmem, 512);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { init_bar(bars.full + s, 1); init_bar(bars.empty + s, empties); }
    for (int g = 0; g < kGroups; ++g) { init_bar(bars.ready + g, 4); init_bar(bars.taken + g, 1); }
    init_bar(&bars.drain, 1);
    for (int b = 0; b < 2; ++b) { init_bar(bars.acc_full + b, 1); init_bar(bars.acc_empty + b, kWarps); }
    fence_bars();
    bars.failed = 0;
  }
  fence_before();
  __syncthreads();
  fence_after();
}

// The stages' loads, by a warp: `boxes` of dy, EACH columns apart, then the codes.
template <int STAGES, int EACH>
__device__ __forceinline__ void load_stages(const CUtensorMap* dy, const CUtensorMap* codes, Bars& bars, uint32_t ring, uint32_t stage_bytes, uint32_t codes_at, int boxes, const Place& at,
                                            uint32_t& left, int& s, uint32_t& round) {
  const bool mine = elected() != 0u;
  if (mine) {
    prefetch_map(dy);
    prefetch_map(codes);
  }
  __syncwarp();
  for (int i = 0; i < at.stages; ++i) {
    if (round > 0) wait_bar(bars.empty + s, (round - 1) & 1, left);
    const bool go = mine && left != 0u;
    const uint32_t stage = ring + (uint32_t)s * stage_bytes, bar = smem_u32(bars.full + s);
    const int row = (int)(at.row0 + (int64_t)i * kRows);
    expect_if(go, bars.full + s, (uint32_t)(boxes + 1) * kBox);
    for (int b = 0; b < boxes; ++b) tma_load(go, dy, stage + (uint32_t)b * kBox, bar, at.n0 + b * EACH, row);
    tma_load(go, codes, stage + codes_at, bar, at.group * kGroup, row);
    if (++s == STAGES) { s = 0; ++round; }
  }
}

// All roles are done; whether a wait of one of them has run out.
__device__ __forceinline__ bool settle(Bars& bars, uint32_t left) {
  if (left == 0u) bars.failed = 1;
  fence_before();
  __syncthreads();
  fence_after();
  return bars.failed != 0;
}
// The way out, after the last read of TMEM: when a wait has run out, what was issued is waited for (bounded) before TMEM is freed.
template <int STAGES>
__device__ __forceinline__ void leave(const Params& p, Bars& bars, bool lost, int s, uint32_t round) {
  const int wid = threadIdx.x >> 5;
  if (lost && p.tries != 0u) {
    uint32_t left = p.tries;
    if (wid == kWarps) {
      for (int q = 0; q < STAGES; ++q) {
        const uint32_t uses = round + (q < s ? 1u : 0u);
        if (uses > 0) wait_bar(bars.full + q, (uses - 1) & 1, left);
      }
    } else if (wid == kWarps + 1) {
      const bool mine = elected() != 0u;
      commit(mine, &bars.drain);
      wait_bar(&bars.drain, 0, left);
    }
  }
  fence_before();
  __syncthreads();
  if (wid == kWarps + 1) {
    fence_after();
    free_tmem(bars.tmem, 512);
  }
  if (threadIdx.x == 0 && lost) report_wait(p.error, 8);
}

// ---------------------------------------------------------------- bfloat16: x decoded, in TMEM; dy as it is
constexpr int kWide = 256;                                           // columns of dy in a tile
constexpr int kWideTaken = 64;                                       // stages between two takings out
constexpr uint32_t kWideStage = (kWide / 64 + 1) * kBox;             // four boxes of 64 columns, and the codes
constexpr int kWideStages = 7, kWideSmem = kWideStages * kWideStage + 32 * 32 * kWarps * 4 + 1024;  // and sums that have been taken out

__global__ void __launch_bounds__(kThreads, 1) rows_kernel(const __grid_constant__ CUtensorMap dy, const __grid_constant__ CUtensorMap codes, const __grid_constant__ Params p) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ Bars bars;
  __shared__ __align__(16) float scales_s[kWarps][64];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  const Place at(p, kWide);
  const int cols = min(kWide, p.n - at.n0), boxes = (cols + 63) / 64;
  uint32_t left = p.tries;
  int s = 0;
  uint32_t round = 0;
  begin(bars, 5);  // a stage is free when its MMAs are done and its group's warps have read it
  const uint32_t tmem = bars.tmem, ring = smem_u32(smem), a_tmem = tmem + kWide;
  const int quarter = wid & 3, set = wid >> 2, takes = (at.stages + kWideTaken - 1) / kWideTaken;
  // What has been taken out of a group's 64 columns of the accumulators: 32 in shared memory, four for all threads side by side, and 32 in the columns of TMEM that are left.
  const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)set * 64, held = a_tmem + kGroups * 32 + ((uint32_t)(quarter * 32) << 16) + (uint32_t)set * 32;
  float4* const sums = reinterpret_cast<float4*>(smem + kWideStages * kWideStage) + tid;
  f32x2 of_bias = 0ull;
  dependency_wait();
  release_dependents();

  if (wid == kWarps) {
    load_stages<kWideStages, 64>(&dy, &codes, bars, ring, kWideStage, (kWide / 64) * kBox, boxes, at, left, s, round);
  } else if (wid == kWarps + 1) {
    // ================= MMAs
    const bool mine = elected() != 0u;
    const uint32_t idesc = instruction(kSumF32, kFormatBf16, 128, (uint32_t)(cols + 15) / 16 * 16) | kTurnedB, b_low = desc_low(ring, kBox);
    for (int i = 0; i < at.stages; ++i) {
      const int slot = i % kGroups, t = i / kWideTaken;
      const bool starts = i % kWideTaken == 0;
      if (starts && t > 0) wait_bar(bars.acc_empty, (t - 1) & 1, left);
      wait_bar(bars.full + s, round & 1, left);
      wait_bar(bars.ready + slot, (i / kGroups) & 1, left);
      fence_after();
      const bool go = mine && left != 0u;
      const uint32_t b = b_low + (uint32_t)s * (kWideStage >> 4), a = a_tmem + (uint32_t)slot * 32;
#pragma unroll
      for (uint32_t q = 0; q < kRows / 16; ++q) {
        mma_f16_tmem(go, tmem, a + 8 * q, desc(b + q * kStepTurned), idesc, !starts || q != 0);
        mma_f16_tmem(go, tmem, a + 16 + 8 * q, desc(b + q * kStepTurned), idesc, true);
      }
      commit(go, bars.empty + s);
      commit(go, bars.taken + slot);
      if (i % kWideTaken == kWideTaken - 1 || i == at.stages - 1) commit(go, bars.acc_full);
      if (++s == kWideStages) { s = 0; ++round; }
    }
  } else {
    const auto take = [&](int t) {  // sums out of TMEM
      wait_bar(bars.acc_full, t & 1, left);
      fence_after();
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        uint32_t r[32];
        tmem_ld32(acc + 32 * part, r);
        tmem_wait(r);
        if (part == 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float4 v = t > 0 ? sums[j * 32 * kWarps] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            v.x += __uint_as_float(r[4 * j]); v.y += __uint_as_float(r[4 * j + 1]); v.z += __uint_as_float(r[4 * j + 2]); v.w += __uint_as_float(r[4 * j + 3]);
            sums[j * 32 * kWarps] = v;
          }
        } else {
          if (t > 0) {
            uint32_t before[32];
            tmem_ld32(held, before);
            tmem_wait(before);
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(before[j]));
          }
          tmem_st32(held, r);
        }
      }
      tmem_st_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(bars.acc_empty);
    };
    // ================= x as two bfloat16 numbers: a column a thread, a stage a group
    const int c = quarter * 32 + lane;
    uint32_t column[8];  // of row j of eight, in the 128-byte swizzle
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) column[j] = ring + (kWide / 64) * kBox + j * 128 + ((((uint32_t)c >> 4) ^ j) << 4) + (c & 15);
    const uint32_t to = a_tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)set * 32;
    Scales scale;
    scale.fetch(p, at.row0, at.rows, set, at.group);
    int use = 0, taken = 0;
    for (int i = set; i < at.stages; i += kGroups, ++use) {
      s = i % kWideStages;
      scale.tell(scales_s[wid]);
      scale.fetch(p, at.row0, at.rows, i + kGroups, at.group);
      wait_bar(bars.full + s, (uint32_t)(i / kWideStages) & 1, left);
      const uint32_t stage = (uint32_t)s * kWideStage;
      uint32_t q[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) q[r] = lds_u8(column[r & 7] + stage + (uint32_t)(r >> 3) * 1024);
      if (at.group == 0) {  // two columns of dy a thread, over the stage's rows
        const uint32_t box = ring + stage + (uint32_t)quarter * kBox;
        if (quarter < boxes) {
#pragma unroll 8
          for (uint32_t r = 0; r < kRows; ++r) {
            const uint32_t w = lds_u32(box + r * 128 + ((((uint32_t)lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
            of_bias = plus2(of_bias, pair_of(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)));
          }
        }
      }
      __syncwarp();
      if (lane == 0) arrive(bars.empty + s);
      uint32_t high[16], low[16];
#pragma unroll
      for (int r = 0; r < kRows; r += 4) {
        const float4 step = *reinterpret_cast<const float4*>(&scales_s[wid][r]), base = *reinterpret_cast<const float4*>(&scales_s[wid][32 + r]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f32x2 v = plus2(pair_of(__uint_as_float(q[r + 2 * h] | 0x4B000000u), __uint_as_float(q[r + 2 * h + 1] | 0x4B000000u)), both(-8388608.0f));
          v = fma2(h ? pair_of(step.z, step.w) : pair_of(step.x, step.y), v, h ? pair_of(base.z, base.w) : pair_of(base.x, base.y));
          high[r / 2 + h] = pack_bf16(v);
          low[r / 2 + h] = pack_bf16(less_bf16(v, high[r / 2 + h]));
        }
      }
      if (use > 0) wait_bar(bars.taken + set, (uint32_t)(use - 1) & 1, left);
      fence_after();
      tmem_st16(to, high);
      tmem_st16(to + 16, low);
      tmem_st_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(bars.ready + set);
      // sums of stages that were handed over a round ago
      if ((taken + 1) * kWideTaken <= i) take(taken++);
    }
    while (taken + 1 < takes) take(taken++);
    wait_bar(bars.acc_full, (takes - 1) & 1, left);
  }
  const bool lost = settle(bars, left);
  if (wid < kWarps) {  // a group has 64 columns of dy, a thread a column of x
    const float none = lost ? __int_as_float(0x7fffffff) : 0.0f;
    const int x_col = at.group * kGroup + quarter * 32 + lane;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int c0 = set * 64 + 32 * part;
      if (c0 >= cols) break;
      uint32_t r[32];
      tmem_ld32(acc + 32 * part, r);
      tmem_wait(r);
      if (takes > 1) {  // and what has been taken out before
        if (part == 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 v = sums[j * 32 * kWarps];
            r[4 * j] = __float_as_uint(__uint_as_float(r[4 * j]) + v.x);
            r[4 * j + 1] = __float_as_uint(__uint_as_float(r[4 * j + 1]) + v.y);
            r[4 * j + 2] = __float_as_uint(__uint_as_float(r[4 * j + 2]) + v.z);
            r[4 * j + 3] = __float_as_uint(__uint_as_float(r[4 * j + 3]) + v.w);
          }
        } else {
          uint32_t before[32];
          tmem_ld32(held, before);
          tmem_wait(before);
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) + __uint_as_float(before[j]));
        }
      }
      if (at.part >= 0) {
        float4* const out = reinterpret_cast<float4*>(p.part) + (int64_t)at.part * (kWide * 128 / 4) + c0 / 4 * 128 + quarter * 32 + lane;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          out[j * 128] = make_float4(__uint_as_float(r[4 * j]) + none, __uint_as_float(r[4 * j + 1]) + none, __uint_as_float(r[4 * j + 2]) + none, __uint_as_float(r[4 * j + 3]) + none);
      } else if (x_col < p.k) {
        __nv_bfloat16* const out = (__nv_bfloat16*)p.dw + (int64_t)(at.n0 + c0) * p.k + x_col;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c0 + j < cols) out[(int64_t)j * p.k] = __float2bfloat16_rn(__uint_as_float(r[j]) + none);
      }
    }
  }
  leave<kWideStages>(p, bars, lost, s, round);
  if (at.group != 0) return;
  float* const columns = reinterpret_cast<float*>(smem);  // [group][256]: the ring is free
  if (wid < kWarps) *reinterpret_cast<f32x2*>(columns + set * kWide + quarter * 64 + 2 * lane) = of_bias;
  __syncthreads();
  if (tid < cols) {
    float sum = lost ? __int_as_float(0x7fffffff) : 0.0f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) sum += columns[g * kWide + tid];
    if (at.part >= 0) p.part_db[(int64_t)at.split * p.n_tiles * kWide + at.n0 + tid] = sum;
    else ((__nv_bfloat16*)p.db)[at.n0 + tid] = __float2bfloat16_rn(sum);
  }
}

// ---------------------------------------------------------------- float32, float16: dy times the step, in TMEM; the codes as they are
constexpr int kTile = 128;                     // columns of dy in a tile
constexpr uint32_t kCodesBytes = 2 * kBox;     // a stage's codes as bfloat16

// kTaken: stages between two takings out
template <typename T> struct Kind;
template <> struct Kind<float> {
  static constexpr int kPieces = 3, kTaken = 8, kEach = 32;
  static constexpr uint32_t kStage = 5 * kBox;
};
template <> struct Kind<__half> {
  static constexpr int kPieces = 2, kTaken = 32, kEach = 64;
  static constexpr uint32_t kStage = 3 * kBox;
};
template <typename T> constexpr int kTileSmem = kStages * Kind<T>::kStage + kGroups * kCodesBytes + 1024;

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) scaled_kernel(const __grid_constant__ CUtensorMap dy, const __grid_constant__ CUtensorMap codes, const __grid_constant__ Params p) {
  constexpr int kPieces = Kind<T>::kPieces, kTaken = Kind<T>::kTaken, kEach = Kind<T>::kEach;
  constexpr uint32_t kStage = Kind<T>::kStage, kCodesAt = kStage - kBox;
  extern __shared__ unsigned char smem_raw[];
  __shared__ Bars bars;
  __shared__ __align__(16) float scales_s[kWarps][96];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, wid = tid >> 5, lane = tid & 31;
  const Place at(p, kTile);
  const int cols = min(kTile, p.n - at.n0), boxes = (cols + kEach - 1) / kEach, takes = (at.stages + kTaken - 1) / kTaken;
  uint32_t left = p.tries;
  int s = 0;
  uint32_t round = 0;
  begin(bars, 4);  // a stage is free when its group's warps have read it
  const uint32_t tmem = bars.tmem, ring = smem_u32(smem), q_ring = ring + kStages * kStage, a_tmem = tmem + 2 * kTile;
  const int quarter = wid & 3, set = wid >> 2;
  f32x2 sum[16], of_base = 0ull, of_bias = 0ull;
#pragma unroll
  for (int j = 0; j < 16; ++j) sum[j] = 0ull;
  dependency_wait();
  release_dependents();

  if (wid == kWarps) {
    load_stages<kStages, kEach>(&dy, &codes, bars, ring, kStage, kCodesAt, boxes, at, left, s, round);
  } else if (wid == kWarps + 1) {
    // ================= MMAs
    const bool mine = elected() != 0u;
    const uint32_t idesc = instruction(kSumF32, kFormatBf16, kTile, kTile) | kTurnedB, b_low = desc_low(q_ring, kBox);
    for (int i = 0; i < at.stages; ++i) {
      const int slot = i % kGroups, t = i / kTaken, in_take = i % kTaken;
      const uint32_t acc = tmem + (uint32_t)(t & 1) * kTile;
      if (in_take == 0 && t >= 2) wait_bar(bars.acc_empty + (t & 1), ((t >> 1) - 1) & 1, left);
      wait_bar(bars.ready + slot, (i / kGroups) & 1, left);
      fence_after();
      const bool go = mine && left != 0u;
      const uint32_t b = b_low + (uint32_t)slot * (kCodesBytes >> 4), a = a_tmem + (uint32_t)slot * (16 * kPieces);
#pragma unroll
      for (uint32_t q = 0; q < kRows / 16; ++q)
#pragma unroll
        for (int piece = kPieces - 1; piece >= 0; --piece)  // the small ones first
          mma_f16_tmem(go, acc, a + 16 * piece + 8 * q, desc(b + q * kStepTurned), idesc, in_take != 0 || q != 0 || piece != kPieces - 1);
      commit(go, bars.taken + slot);
      if (in_take == kTaken - 1 || i == at.stages - 1) commit(go, bars.acc_full + (t & 1));
    }
  } else {
    const auto take = [&](int t) {  // sums out of TMEM: a group has 32 columns of the codes, a thread a column of dy
      wait_bar(bars.acc_full + (t & 1), (t >> 1) & 1, left);
      fence_after();
      uint32_t r[32];
      tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)((t & 1) * kTile + set * 32), r);
      tmem_wait(r);
#pragma unroll
      for (int j = 0; j < 16; ++j) sum[j] = plus2(sum[j], pair_of(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])));
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(bars.acc_empty + (t & 1));
    };
    // ================= dy times the step as bfloat16 numbers, a column a thread, a stage a group
    const int c = quarter * 32 + lane;
    uint32_t column[8];  // of row j of eight, in the 128-byte swizzle
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      if constexpr (sizeof(T) == 4) column[j] = ring + (uint32_t)quarter * kBox + j * 128 + ((((uint32_t)lane >> 2) ^ j) << 4) + (lane & 3) * 4;
      else column[j] = ring + (uint32_t)(quarter >> 1) * kBox + j * 128 + (((((uint32_t)c & 63) >> 3) ^ j) << 4) + (c & 7) * 2;
    }
    // and codes: 32 of a row a thread
    const uint32_t q_row = (uint32_t)(tid & 127) >> 2, q_part = tid & 3;
    const uint32_t to = a_tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)set * (16 * kPieces);
    Scales scale;
    scale.fetch(p, at.row0, at.rows, set, at.group);
    int use = 0, taken = 0;
    for (int i = set; i < at.stages; i += kGroups, ++use) {
      s = i % kStages;
      scale.tell_about_zero(scales_s[wid]);
      scale.fetch(p, at.row0, at.rows, i + kGroups, at.group);
      wait_bar(bars.full + s, (uint32_t)(i / kStages) & 1, left);
      const uint32_t stage = (uint32_t)s * kStage;
      const bool mine = quarter * 32 < cols;  // (behind them nothing was loaded)
      // 16 rows at a time: more did not fit into the registers beside the sums
#pragma unroll
      for (uint32_t half = 0; half < 2; ++half) {
        f32x2 d[8];
        const uint32_t from = stage + half * 2048;
        if (mine) {
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            const uint32_t even = column[r & 7] + from + (uint32_t)(r >> 3) * 1024, odd = column[(r + 1) & 7] + from + (uint32_t)(r >> 3) * 1024;
            if constexpr (sizeof(T) == 4) d[r / 2] = pair_of(__uint_as_float(lds_u32(even)), __uint_as_float(lds_u32(odd)));
            else d[r / 2] = pair_of(__half2float(__ushort_as_half((unsigned short)lds_u16(even))), __half2float(__ushort_as_half((unsigned short)lds_u16(odd))));
          }
        } else {
#pragma unroll
          for (int r = 0; r < 8; ++r) d[r] = 0ull;
        }
        if (at.group == 0) {
#pragma unroll
          for (int r = 0; r < 8; ++r) of_bias = plus2(of_bias, d[r]);
        }
        const float* const step_of = scales_s[wid] + half * 16;
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
          const float4 step = *reinterpret_cast<const float4*>(step_of + r), base = *reinterpret_cast<const float4*>(step_of + 32 + r);
          of_base = fma2(pair_of(base.x, base.y), d[r / 2], of_base);
          of_base = fma2(pair_of(base.z, base.w), d[r / 2 + 1], of_base);
          d[r / 2] = mul2(pair_of(step.x, step.y), d[r / 2]);
          d[r / 2 + 1] = mul2(pair_of(step.z, step.w), d[r / 2 + 1]);
        }
#pragma unroll
        for (int piece = 0; piece < kPieces; ++piece) {
          uint32_t w[8];
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            w[r] = kPieces == 3 ? cut_bf16(d[r]) : pack_bf16(d[r]);  // (of three, what the last leaves is nothing)
            if (piece + 1 < kPieces) d[r] = less_bf16(d[r], w[r]);
          }
          if (piece == 0 && half == 0) {  // what the group handed over a round ago has been used
            if (use > 0) wait_bar(bars.taken + set, (uint32_t)(use - 1) & 1, left);
            fence_after();
          }
          tmem_st8(to + 16 * piece + 8 * half, w);
        }
      }
      const f32x2 zero = both(-scales_s[wid][64 + q_row]);
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {  // 16 codes
        const uint4 q = lds_u128(ring + stage + kCodesAt + q_row * 128 + (((q_part * 2 + h) ^ (q_row & 7)) << 4));
        const uint32_t box = q_ring + (uint32_t)set * kCodesBytes + (q_part >> 1) * kBox + q_row * 128, first = (q_part & 1) * 4 + 2 * h;
        f32x2 a[2], b[2];
        ckpt::numbers_of(q.x, zero, a);
        ckpt::numbers_of(q.y, zero, b);
        sts_u128(box + ((first ^ (q_row & 7)) << 4), pack_bf16(a[0]), pack_bf16(a[1]), pack_bf16(b[0]), pack_bf16(b[1]));
        ckpt::numbers_of(q.z, zero, a);
        ckpt::numbers_of(q.w, zero, b);
        sts_u128(box + (((first + 1) ^ (q_row & 7)) << 4), pack_bf16(a[0]), pack_bf16(a[1]), pack_bf16(b[0]), pack_bf16(b[1]));
      }
      __syncwarp();
      if (lane == 0) arrive(bars.empty + s);
      tmem_st_wait();
      fence_async();
      fence_before();
      __syncwarp();
      if (lane == 0) arrive(bars.ready + set);
      // sums of stages that were handed over a round ago
      if ((taken + 1) * kTaken <= i) take(taken++);
    }
    while (taken < takes) take(taken++);
  }
  const bool lost = settle(bars, left);
  leave<kStages>(p, bars, lost, s, round);
  float(*const columns)[2][kTile] = reinterpret_cast<float(*)[2][kTile]>(smem);  // [group]: the ring is free, and behind them for the tile
  if (wid < kWarps) {
    columns[set][0][quarter * 32 + lane] = lo32(of_base) + hi32(of_base);
    columns[set][1][quarter * 32 + lane] = lo32(of_bias) + hi32(of_bias);
  }
  __syncthreads();
  if (wid >= kWarps) return;
  const int i = quarter * 32 + lane;
  float more = lost ? __int_as_float(0x7fffffff) : 0.0f, bias = more;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    more += columns[g][0][i];
    bias += columns[g][1][i];
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) sum[j] = plus2(sum[j], both(more));
  if (at.part >= 0) {
    ulonglong2* const out = reinterpret_cast<ulonglong2*>(p.part) + (int64_t)at.part * (kTile * kTile / 4) + set * 8 * kTile + i;
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j * kTile] = make_ulonglong2(sum[2 * j], sum[2 * j + 1]);
    if (at.group == 0 && set == 0) p.part_db[(int64_t)at.split * p.n_tiles * kTile + at.n0 + i] = bias;
    return;
  }
  if (at.group == 0 && set == 0 && i < cols) ((T*)p.db)[at.n0 + i] = from_float<T>(bias);
  // Rows of the result are written by whole warps, two columns a lane.  (By the threads that have them, a row each, 4 x 3634 x 1860 float16 took 71 us instead of 17.)
  constexpr int kPitch = kTile + 2;  // (two columns at a time, rows on other banks)
  float* const tile = reinterpret_cast<float*>(smem + 8192);
#pragma unroll
  for (int j = 0; j < 16; ++j) *reinterpret_cast<f32x2*>(tile + i * kPitch + set * 32 + 2 * j) = sum[j];
  asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");  // (the two warps that load and issue are gone)
  const int width = min(kGroup, p.k - at.group * kGroup);
  const bool pairs = (p.k & 1) == 0 && (reinterpret_cast<uintptr_t>(p.dw) & (2 * sizeof(T) - 1)) == 0;
  for (int r = wid; r < cols; r += kWarps) {
    T* const out = (T*)p.dw + (int64_t)(at.n0 + r) * p.k + at.group * kGroup;
#pragma unroll
    for (int c = 2 * lane; c < kTile; c += 64) {
      const float2 v = *reinterpret_cast<const float2*>(tile + r * kPitch + c);
      struct alignas(2 * sizeof(T)) Two { T a, b; };
      if (pairs && c + 1 < width) {
        *reinterpret_cast<Two*>(out + c) = Two{from_float<T>(v.x), from_float<T>(v.y)};
      } else {
        if (c < width) out[c] = from_float<T>(v.x);
        if (c + 1 < width) out[c + 1] = from_float<T>(v.y);
      }
    }
  }
}

// Adds the parts up: 32 lanes and four columns of TMEM to a CTA, every 16th part (or as many as there are) to a
// warp.  Behind the tiles' CTAs those of db (where no tile is whole: otherwise those of the first group are).  The lanes are columns
// of x (bfloat16) or of dy.
constexpr int kJoinWarps = 16;
template <typename T>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ Params p) {
  constexpr bool kOfX = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kColumns = kOfX ? kWide : kTile, kPerTile = kColumns, kQuads = kColumns * 128 / 4;
  __shared__ float4 of[kJoinWarps][33];
  dependency_wait();
  release_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, tiles = p.rest;
  if ((int)blockIdx.x >= tiles * kPerTile) {
    const int i = ((int)blockIdx.x - tiles * kPerTile) * 32 + lane;
    float sum = 0.0f;
    for (int s = warp; s < p.splits; s += warps) sum += p.part_db[(int64_t)s * p.n_tiles * kColumns + i];
    of[warp][lane].x = sum;
    __syncthreads();
    if (warp != 0 || i >= p.n) return;
    sum = 0.0f;
    for (int w = 0; w < warps; ++w) sum += of[w][lane].x;
    ((T*)p.db)[i] = from_float<T>(sum);
    return;
  }
  const int tile = blockIdx.x / kPerTile, rest = blockIdx.x % kPerTile, quad = rest / 4, i = rest % 4 * 32 + lane;
  const float4* const from = reinterpret_cast<const float4*>(p.part) + (int64_t)tile * kQuads + quad * 128 + i;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 10
  for (int s = warp; s < p.splits; s += warps) {
    const float4 v = from[(int64_t)s * tiles * kQuads];
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  }
  of[warp][lane] = sum;
  __syncthreads();
  const int across = (p.whole + tile) % p.n_tiles * kColumns, down = (p.whole + tile) / p.n_tiles * kGroup;
  const int n = across + (kOfX ? quad * 4 : i), col = down + (kOfX ? i : quad * 4);
  if (warp != 0 || n >= p.n || col >= p.k) return;
  sum = of[0][lane];
  for (int w = 1; w < warps; ++w) {
    const float4 v = of[w][lane];
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  }
  T* const to = (T*)p.dw + (int64_t)n * p.k + col;
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if ((kOfX ? n : col) + e < (kOfX ? p.n : p.k)) to[kOfX ? (int64_t)e * p.k : e] = from_float<T>(v[e]);
}

// Copies dy to rows that start on 16 bytes, where TMA can read them.
template <typename T>
__global__ void __launch_bounds__(256) align_kernel(const T* __restrict__ src, int64_t ld, int64_t n, T* __restrict__ dst, int64_t aligned_ld, int64_t m) {
  dependency_wait();
  release_dependents();
  const int64_t total = m * n;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / n;
    dst[row * aligned_ld + (i - row * n)] = src[row * ld + (i - row * n)];
  }
}

struct Plan {
  int columns, n_tiles, k_tiles, splits, whole, rest;
  int64_t split_rows, part_bytes, sum_bytes, copy_ld, bytes;  // copy_ld: 0 where dy can be read where it is
};

// How many ways the rows are split: the choice of least time, in cycles: a stage takes an SM 560 (bfloat16: its MMAs), 1200 (float32) or 900 (float16: what
// the groups do for it); together the SMs get no more than 3500 bytes a cycle; a tile's start and end 4000, the parts' way through L2 and back 4000 bytes a
// cycle for all SMs, and the launch that adds them up 4000.  With more tiles than SMs those that fill the SMs are left whole and the rows of the others split, where
// that is an eighth less: 196 tiles, 16,384 x 1700 x 1700 float32 509 us without and 370 so; 152 tiles, 8192 x 2048 x 2368 bfloat16 188 and 137; but 256 tiles,
// 16,384 x 2048 x 4096 bfloat16 416 and 429 (SMs that wait leave the others power; both before its sums were taken out).
static Plan plan(const void* dy, int64_t ldy, int dtype, int64_t m, int64_t n, int64_t k) {
  Plan p{};
  const int64_t item = dtype_size(dtype);
  p.columns = dtype == F2C_BF16 ? kWide : kTile;
  p.n_tiles = (int)ceil_div(n, p.columns);
  p.k_tiles = (int)ceil_div(k, kGroup);
  const int64_t tiles = (int64_t)p.n_tiles * p.k_tiles, stages = ceil_div(m, kRows), tile_bytes = (int64_t)p.columns * 128 * 4;
  const int64_t first = ceil_div(m, kMaxSplitRows);
  int64_t least = INT64_MAX;
  const auto consider = [&](int64_t whole, int64_t s) {
    const int64_t each = ceil_div(stages, s), rest = tiles - whole;
    if (s > first && ceil_div(stages, each) != s) return;  // (the last ones would have none)
    const int64_t stage_bytes = kRows * ((int64_t)p.columns * item / p.k_tiles + 128 / p.n_tiles);
    const int64_t stage = std::max<int64_t>(dtype == F2C_BF16 ? 560 : dtype == F2C_F32 ? 1200 : 900, std::min<int64_t>(whole + rest * s, kSmCount) * stage_bytes / 3500);
    const int64_t cycles = whole / kSmCount * (stages * stage + 4000) + ceil_div(rest * s, kSmCount) * (each * stage + 4000) + (s > 1 ? 4000 + rest * s * 2 * tile_bytes / 4000 : 0);
    const int64_t cost = whole > 0 ? cycles + cycles / 8 : cycles;
    if (cost >= least) return;
    least = cost;
    p.split_rows = each * kRows;
    p.splits = (int)ceil_div(stages, each);
    p.whole = (int)whole;
    p.rest = (int)rest;
  };
  for (int64_t s = first; s <= std::min<int64_t>(stages, std::max<int64_t>(first, kSmCount)) && (s == first || tiles * s <= 2 * kSmCount); ++s) consider(0, s);
  const int64_t whole = tiles / kSmCount * kSmCount;
  if (first == 1 && whole >= p.n_tiles && whole < tiles)
    for (int64_t s = 2; s <= stages && (tiles - whole) * s <= 4 * kSmCount; ++s) consider(whole, s);
  if (p.splits > 1) {
    p.part_bytes = (int64_t)p.rest * p.splits * tile_bytes;
    p.sum_bytes = p.whole > 0 ? 0 : ceil_div((int64_t)p.splits * p.n_tiles * p.columns * 4, 256) * 256;
  }
  p.bytes = p.part_bytes + p.sum_bytes;
  if (!aligned(dy, 16) || (m > 1 && ldy * item % 16 != 0)) {
    p.copy_ld = ceil_div(n * item, 16) * 16 / item;
    p.bytes += ceil_div(m * p.copy_ld * item, 256) * 256;
  }
  return p;
}

// A map of a row-major matrix for boxes of kRows rows of 128 bytes.
static bool rows_map(CUtensorMap* map, const void* base, int64_t item, int64_t m, int64_t cols, int64_t ld) {
  // (a lone row may have any stride)
  const int64_t row_bytes = m > 1 ? ld * item : ceil_div(cols * item, 16) * 16;
  return make_map(map, base, (int)item, m, cols, row_bytes, kRows);
}

template <typename T>
static int run(const char* op, const CUtensorMap& dy, const CUtensorMap& codes, const Params& p, const Plan& how, cudaStream_t st) {
  const dim3 grid((unsigned)(how.whole + how.rest * how.splits));
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    if (const int rc = allow_smem(op, (const void*)rows_kernel, kWideSmem)) return rc;
    launch_dependent(rows_kernel, grid, kThreads, kWideSmem, st, dy, codes, p);
  } else {
    if (const int rc = allow_smem(op, (const void*)scaled_kernel<T>, kTileSmem<T>)) return rc;
    launch_dependent(scaled_kernel<T>, grid, kThreads, kTileSmem<T>, st, dy, codes, p);
  }
  if (how.splits > 1)
    launch_dependent(join_kernel<T>, dim3((unsigned)(how.rest * how.columns + (how.whole > 0 ? 0 : how.n_tiles * how.columns / 32))), 32 * std::min(kJoinWarps, how.splits), 0, st, p);
  return check_launch(op);
}

static bool too_large(int64_t m, int64_t n, int64_t k) { return m >= ckpt::kMaxRows - kRows * kStages || n > (1 << 17) || k > (1 << 17); }

}  // namespace wg
}  // namespace f2c

using namespace f2c;

extern "C" int64_t f2c_checkpoint_weight_grad_workspace(const void* dy, int64_t ldy, int dtype, int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || !is_float_dtype(dtype) || wg::too_large(m, n, k)) return 0;
  return wg::plan(dy, ldy, dtype, m, n, k).bytes;
}

extern "C" int f2c_checkpoint_weight_grad(const void* dy, int64_t ldy, int dtype, const uint8_t* codes, int64_t ldq, const float* scales, int64_t m, int64_t n, int64_t k, void* dw,
                                          void* db, int flags, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* op = "checkpoint_weight_grad";
  if (const int rc = ckpt::check_sizes(op, dtype, m, k)) return rc;
  F2C_REQUIRE(n >= 0, F2C_ERR_INVALID, "%s: negative size", op);
  F2C_REQUIRE(!wg::too_large(m, n, k), F2C_ERR_LIMIT, "%s: 2^31 - 256 rows, or more than 2^17 columns", op);
  F2C_REQUIRE((flags & ~F2C_NO_WAITS) == 0, F2C_ERR_INVALID, "%s: unknown flags", op);
  if (const int rc = ckpt::check_codes(op, codes, ldq, scales, m, k)) return rc;
  if (n == 0) return F2C_OK;
  F2C_REQUIRE(db && (dw || k == 0), F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(m == 0 || dy, F2C_ERR_INVALID, "%s: null pointer", op);
  F2C_REQUIRE(m <= 1 || ldy >= n, F2C_ERR_INVALID, "%s: a row stride is smaller than the row", op);
  F2C_REQUIRE(k > 0 || m == 0, F2C_ERR_INVALID, "%s: no columns", op);
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t item = dtype_size(dtype);
  if (m == 0) {
    cudaError_t e = cudaMemsetAsync(db, 0, (size_t)(n * item), st);
    if (e == cudaSuccess && k > 0) e = cudaMemsetAsync(dw, 0, (size_t)(n * k * item), st);
    if (e != cudaSuccess) return set_error(F2C_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
    return F2C_OK;
  }
  const wg::Plan how = wg::plan(dy, ldy, dtype, m, n, k);
  F2C_REQUIRE(how.bytes == 0 || (workspace && workspace_bytes >= how.bytes && aligned(workspace, 256)), F2C_ERR_INVALID,
              "%s: the workspace must have %lld bytes, 256-byte aligned", op, (long long)how.bytes);
  char* const ws = (char*)workspace;
  if (how.copy_ld != 0) {
    char* const copy = ws + how.part_bytes + how.sum_bytes;
    const dim3 grid((unsigned)std::min<int64_t>(ceil_div(m * n, 256), 16 * kSmCount));
    if (item == 4) launch_dependent(wg::align_kernel<uint32_t>, grid, 256, 0, st, (const uint32_t*)dy, ldy, n, (uint32_t*)copy, how.copy_ld, m);
    else launch_dependent(wg::align_kernel<uint16_t>, grid, 256, 0, st, (const uint16_t*)dy, ldy, n, (uint16_t*)copy, how.copy_ld, m);
    dy = copy;
    ldy = how.copy_ld;
  }
  CUtensorMap maps[2] = {};
  F2C_REQUIRE(wg::rows_map(maps, dy, item, m, n, ldy) && wg::rows_map(maps + 1, codes, 1, m, k, ldq), F2C_ERR_CUDA, "%s: tensor map", op);
  const wg::Params p{scales, ceil_div(k, ckpt::kGroup), m, (int)n, (int)k, how.n_tiles, how.splits, how.whole, how.rest, how.split_rows, dw, db, (float*)ws, (float*)(ws + how.part_bytes),
                     (flags & F2C_NO_WAITS) ? 0u : t5::kWaitLimit, stream_error_word()};
  if (dtype == F2C_F32) return wg::run<float>(op, maps[0], maps[1], p, how, st);
  if (dtype == F2C_F16) return wg::run<__half>(op, maps[0], maps[1], p, how, st);
  return wg::run<__nv_bfloat16>(op, maps[0], maps[1], p, how, st);
}
