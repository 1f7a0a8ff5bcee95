// Thin wrappers of the sm_100a instructions that the attention kernels for long segments use: matrix
// products into tensor memory (tcgen05), tensor memory loads and stores, and mbarriers with bounded waits.
//
// Operand tiles in shared memory are blocks of 64 columns (128 bytes) by any number of rows, 128 bytes from
// row to row, their 16-byte pieces swizzled by the row (piece ^ row % 8), at 1024-byte boundaries.  Read
// with the contraction along the columns ("by columns") or along the rows ("by rows") the same image
// serves as either kind of operand:
//   by columns: 8-row groups 1024 bytes apart; 16 columns further on are 32 bytes further on;
//   by rows   : 64-column blocks `block` bytes apart, 8-row groups 1024 bytes apart; 16 rows are 2048 bytes.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "vector_io.cuh"

namespace texb {
namespace t5 {

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

// ---- mbarriers ---------------------------------------------------------------------------------------
__device__ __forceinline__ void barrier_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// One arrival for the whole (converged) warp, behind what all its lanes did: 32 arrivals at one word are done one
// after the other, and the warp's next wait queues behind them.
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) barrier_arrive(bar);
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}

// Waits, for a bounded number of polls, until the phase of that parity is complete.  When the polls run out,
// or another thread's have (`*dead`), it returns all the same: the kernel then runs to its end on whatever its
// memory holds, every later wait returning at once, counts the event (texb_device_status, wait_timeouts) and
// returns, instead of hanging.
constexpr int kPolls = 1 << 20;
__device__ __forceinline__ void barrier_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
  if (barrier_try(bar, parity)) return;
  for (int i = 0; i < kPolls; ++i) {
    if (barrier_try(bar, parity)) return;
    if (*dead) return;
  }
  *dead = 1;
}
// The same by all lanes of a warp, which are together again behind it; what the tensor cores did before the phase
// completed is visible.
__device__ __forceinline__ void warp_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
  barrier_wait(bar, parity, dead);
  __syncwarp();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Also expects `bytes` of copies in this phase.
__device__ __forceinline__ void barrier_arrive_expect(uint32_t bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A box of a three-dimensional tensor (columns, heads, rows) into shared memory; the barrier counts its bytes.
// Places behind the tensor's end read as zeros.  The first column is a multiple of 8 (16 bytes).
__device__ __forceinline__ void copy_box(uint32_t to, const CUtensorMap* map, uint32_t bar, int column, int head, int row) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to),
               "l"(map), "r"(bar), "r"(column), "r"(head), "r"(row) : "memory");
}

// ---- tensor memory -----------------------------------------------------------------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t smem_slot, int columns) {  // one whole warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, int columns) {  // the same warp
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns) : "memory");
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_copies() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 columns of the warp's 32 lanes: lane l of the warp reads lane 32 (warp % 4) + l of tensor memory, which
// the upper half of the address names.
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ---- arithmetic on pairs, and of three -----------------------------------------------------------------
__device__ __forceinline__ float max3(float a, float b, float c) {  // a NaN is passed over, as by fmaxf
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<const unsigned long long&>(a)),
      "l"(reinterpret_cast<const unsigned long long&>(b)), "l"(reinterpret_cast<const unsigned long long&>(c)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<const unsigned long long&>(a)),
      "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<const unsigned long long&>(a)),
      "l"(reinterpret_cast<const unsigned long long&>(b)));
  return d;
}

// ---- matrix products ---------------------------------------------------------------------------------
// Descriptor of an operand tile: swizzle of 128 bytes (2 in the top bits), descriptor version 1, 8-row groups
// 1024 bytes apart.  Only the lower half differs between tiles: address and, read by rows, the distance of
// the 64-column blocks, both in units of 16 bytes.
constexpr uint32_t kOperandUpper = 1024u >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t operand_by_columns(uint32_t addr) { return (addr & 0x3ffffu) >> 4 | 1u << 16; }
__device__ __forceinline__ uint32_t operand_by_rows(uint32_t addr, uint32_t block) {
  return (addr & 0x3ffffu) >> 4 | (block >> 4) << 16;
}
// Instruction descriptor: fp32 sums of products of 16-bit values (both operands of one type), M x N,
// `b_by_rows`: the second operand's contraction runs along the rows of its tile.
template <typename T>
__host__ __device__ constexpr uint32_t instruction(int m, int n, bool b_by_rows) {
  const uint32_t type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return 1u << 4 | type << 7 | type << 10 | (b_by_rows ? 1u << 16 : 0u) | uint32_t(n / 8) << 17 | uint32_t(m / 16) << 24;
}
// One thread; `add` false overwrites the sums.
__device__ __forceinline__ void multiply(uint32_t sums, uint32_t a, uint32_t b, uint32_t instr, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(sums), "r"(a), "r"(b), "r"(instr), "r"(uint32_t(add)),
      "r"(kOperandUpper) : "memory");
}
// First operand from tensor memory: one row per lane, two 16-bit values per column.
__device__ __forceinline__ void multiply_tmem(uint32_t sums, uint32_t a, uint32_t b, uint32_t instr, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tmov.b64 db, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(sums), "r"(a), "r"(b), "r"(instr), "r"(uint32_t(add)),
      "r"(kOperandUpper) : "memory");
}
// The barrier completes a phase when all products that this thread issued are done.
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// sums[128 x n] (+)= rows of tile a times rows of tile b, contraction over DP columns.  Tiles of `rows_a`,
// `rows_b` rows: blocks of 64 columns one after the other.
template <int DP>
__device__ __forceinline__ void multiply_columns(uint32_t sums, uint32_t a, int rows_a, uint32_t b, int rows_b, uint32_t instr) {
  const uint32_t first_a = operand_by_columns(a), first_b = operand_by_columns(b);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k)
    multiply(sums, first_a + (k / 4) * (rows_a * 8) + (k % 4) * 2, first_b + (k / 4) * (rows_b * 8) + (k % 4) * 2, instr, k > 0);
}
// sums[128 x DP] (+)= P (16-bit, tensor memory, 128 x ROWS) times the rows of tile b
template <int ROWS>
__device__ __forceinline__ void multiply_rows(uint32_t sums, uint32_t p, uint32_t b, uint32_t instr, bool add) {
  const uint32_t first_b = operand_by_rows(b, ROWS * 128);
#pragma unroll
  for (int k = 0; k < ROWS / 16; ++k) multiply_tmem(sums, p + k * 8, first_b + k * (2048 >> 4), instr, add || k > 0);
}

// One lane of the (converged) warp, always the same.
__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(on));
  return on != 0;
}

// After a wait that gave up: waits, with a limit, for the products that `issuer` issued, and about a
// millisecond for copies that are still under way, and counts the event.  Called by all threads between two
// barriers.
__device__ __forceinline__ void settle(uint32_t bar, bool issuer, int* counter) {
  if (!issuer) return;
  barrier_init(bar, 1);
  commit(bar);
  for (int p = 0; p < kPolls && !barrier_try(bar, 0); ++p) {}
  for (int p = 0; p < 1000; ++p) __nanosleep(1000);
  atomicAdd(counter, 1);
}

}  // namespace t5
}  // namespace texb
