// 5th-generation tensor cores, TMA and their barriers, as the dense operators use them (int8_mm.cu, newton_schulz.cu).
#pragma once
#include <cuda.h>

#include "common.cuh"

namespace f2c {

int* stream_error_word();

namespace t5 {

constexpr size_t kSmemLimit = 227 * 1024;
// Tries of a wait, and nanoseconds after which one may end; they took 4 us each (a wait that ran out after 2^20: 4.2 s).  The longest wait that can
// end is for the sums of a tile, milliseconds.
constexpr uint32_t kWaitLimit = 1u << 18, kWaitHint = 1000;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ---------------------------------------------------------------- barriers
__device__ __forceinline__ void init_bar(const uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void arrive(const uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
// whether this lane of a whole warp is the one to issue
__device__ __forceinline__ uint32_t elected() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(e));
  return e;
}
__device__ __forceinline__ void expect_if(bool go, const uint64_t* bar, uint32_t bytes) {
  asm volatile("{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %2, 0;\n\t@g mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}\n" ::"r"(smem_u32(bar)),
               "r"(bytes), "r"((uint32_t)go)
               : "memory");
}
__device__ __forceinline__ void fence_bars() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }

// How the roles that issue copies and MMAs are written: whole warps run their loops, whose conditions no wait decides, and `go` - this lane is the
// one that issues, and no wait of the role has run out - is a predicate of every instruction that does something.  Then the compiler keeps
// descriptors and addresses in uniform registers.  (With one thread in a loop that a failed wait leaves, a wait took 180 cycles instead of 60 and an
// MMA 60 to 90 instead of 46: more than the MMA itself up to 128 columns.)

// Whether a wait that has tried goes on: not with the phase complete, and not with kWaitLimit tries `spent` (a number of the wait's own, however many
// waits a long product takes).  One that runs out leaves `left` 0: the role has given up for good, and later waits try once.
__host__ __device__ __forceinline__ bool tries_again(bool done, uint32_t& spent, uint32_t& left) {
  if (done || left == 0u) return false;
  if (++spent < kWaitLimit) return true;
  left = 0u;
  return false;
}
__device__ __forceinline__ void wait_bar(const uint64_t* bar, uint32_t parity, uint32_t& left) {
  const uint32_t at = smem_u32(bar);
  uint32_t done, spent = 0;
  do {
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done) : "r"(at), "r"(parity), "r"(kWaitHint) : "memory");
  } while (tries_again(done != 0u, spent, left));
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// ordinary writes to shared memory, before copies and MMAs that read it
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---------------------------------------------------------------- TMEM
// `columns`: a power of two from 32 to 512.  Where the SM's other CTAs hold too many, the allocation waits for them: none of them waits for this one.
__device__ __forceinline__ void alloc_tmem(uint32_t* at, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(at)), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void free_tmem(uint32_t tmem, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

// The same in both CTAs of a pair, by one warp of each.
__device__ __forceinline__ void alloc_tmem_pair(uint32_t* at, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(at)), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void free_tmem_pair(uint32_t tmem, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

// 32 columns from `taddr` on, of the 32 lanes that the warp owns
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// The reads issued so far are complete; naming the registers keeps their uses behind the wait.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]),
                 "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]),
                 "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
                 "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}

// ---------------------------------------------------------------- MMAs
// Operands in shared memory, 128-byte swizzle, atoms of 8 x 128 bytes that start on 1024.  A descriptor's low word holds the address in 16 bytes, to
// which offsets are added as they are: the thread that issues MMAs has few cycles for each.
//  * along K: row r of 128 bytes at 128 r, 32 bytes of K to an MMA
//  * along M or N, one row for every element of K: K row r of 64 elements at 128 r, the next 64 elements `chunk` bytes further; 16 K rows to an MMA
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t chunk) { return ((addr & 0x3FFFFu) >> 4) | ((chunk >> 4) << 16); }
constexpr uint32_t kChunkAlongK = 16;                                     // (has no meaning there)
constexpr uint32_t kStepAlongK = 32 >> 4, kStepTurned = 16 * 128 >> 4;    // from one MMA's operand to the next
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);    // 1024 bytes from atom to atom, sm_100, 128-byte swizzle
__device__ __forceinline__ uint64_t desc(uint32_t low) { return ((uint64_t)kDescHigh << 32) | low; }

constexpr uint32_t kTurnedA = 1u << 15, kTurnedB = 1u << 16;  // of an instruction: the operand lies along M or N
constexpr uint32_t kFormatF16 = 0, kFormatS8 = 1, kSumF32 = 1, kSumS32 = 2;
__device__ __forceinline__ constexpr uint32_t instruction(uint32_t sum, uint32_t format, uint32_t m, uint32_t n) {
  return (sum << 4) | (format << 7) | (format << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

#define F2C_MMA(name, form, lanes)                                                                                              \
  __device__ __forceinline__ void name(bool go, uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {  \
    asm volatile(                                                                                                              \
        "{\n\t.reg .pred p, g;\n\tsetp.ne.b32 g, %6, 0;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                              \
        "@g tcgen05.mma." form " [%0], %1, %2, %3, {" lanes "}, p;\n\t}\n" ::"r"(d_tmem), "l"(a), "l"(b), "r"(idesc),           \
        "r"((uint32_t)accumulate), "r"(0u), "r"((uint32_t)go)                                                                 \
        : "memory");                                                                                                           \
  }
F2C_MMA(mma_i8, "cta_group::1.kind::i8", "%5, %5, %5, %5")
F2C_MMA(mma_f16, "cta_group::1.kind::f16", "%5, %5, %5, %5")
// over both CTAs of a pair: half of the rows of A and of the columns of B in the shared memory of each, at the same offsets
F2C_MMA(mma_i8_pair, "cta_group::2.kind::i8", "%5, %5, %5, %5, %5, %5, %5, %5")
F2C_MMA(mma_f16_pair, "cta_group::2.kind::f16", "%5, %5, %5, %5, %5, %5, %5, %5")
#undef F2C_MMA

// arrives at the barrier when all MMAs issued so far by this thread are complete
__device__ __forceinline__ void commit(bool go, const uint64_t* bar) {
  asm volatile("{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %1, 0;\n\t"
               "@g tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)), "r"((uint32_t)go)
               : "memory");
}
// the same of the MMAs of a pair, at the barriers of its CTAs in `mask`
__device__ __forceinline__ void commit_pair(bool go, const uint64_t* bar, uint16_t mask = 3) {
  asm volatile("{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %2, 0;\n\t"
               "@g tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}\n" ::"r"(smem_u32(bar)),
               "h"(mask), "r"((uint32_t)go)
               : "memory");
}

// ---------------------------------------------------------------- TMA
__device__ __forceinline__ void tma_load(bool go, const CUtensorMap* map, uint32_t dst, uint32_t bar, int x, int y) {
  asm volatile("{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %5, 0;\n\t"
               "@g cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}\n" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(bar), "r"((uint32_t)go)
               : "memory");
}
__device__ __forceinline__ void tma_load(bool go, const CUtensorMap* map, uint32_t dst, uint32_t bar, int x, int y, int z) {
  asm volatile("{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %6, 0;\n\t"
               "@g cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}\n" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "r"((uint32_t)go)
               : "memory");
}
// The same in a pair of CTAs: `bar`, at which the bytes are counted, is a cluster address and may be the other one's.
__device__ __forceinline__ void tma_load_pair(bool go, const CUtensorMap* map, uint32_t dst, uint32_t bar, int x, int y) {
  asm volatile("{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %5, 0;\n\t"
               "@g cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];\n\t}\n" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(bar), "r"((uint32_t)go)
               : "memory");
}
__device__ __forceinline__ void tma_load_pair(bool go, const CUtensorMap* map, uint32_t dst, uint32_t bar, int x, int y, int z) {
  asm volatile("{\n\t.reg .pred g;\n\tsetp.ne.b32 g, %6, 0;\n\t"
               "@g cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];\n\t}\n" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar), "r"((uint32_t)go)
               : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// ---------------------------------------------------------------- clusters
__device__ __forceinline__ void cluster_barrier() {  // of all threads of the cluster; orders their accesses to its shared memory
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_address(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// Tells nothing but itself (what has been read from TMEM may be written over): released to the cluster, it took 900 cycles.
__device__ __forceinline__ void peer_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void peer_store(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

// Tensor map of a row-major matrix [rows, cols] of `bytes`-byte elements (1, 2, or 4: single precision; 16-byte aligned start and row stride), boxes of box_rows x
// 128 bytes with the 128-byte swizzle, zeros outside the matrix.  False when the driver refuses it.
bool make_map(CUtensorMap* map, const void* base, int bytes, int64_t rows, int64_t cols, int64_t row_bytes, int box_rows);
// The same for a stack of `batch` half-precision matrices, `rows` rows apart.
bool make_stack_map(CUtensorMap* map, const void* base, int64_t batch, int64_t rows, int64_t cols, int64_t row_bytes, int box_rows);

}  // namespace t5
}  // namespace f2c
