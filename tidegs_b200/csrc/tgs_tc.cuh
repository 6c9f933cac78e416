// tcgen05 wrappers (sm_100a, one CTA): tensor memory, matrix instructions on
// bf16 operands in shared memory, and the 128-byte swizzled operand layout.
//
// Operand blocks: [rows][64] bf16, rows of 128 bytes in 1024-byte groups of
// eight, the 16-byte unit u of row r stored at unit u ^ (r % 8). One block
// serves both ways round: with its rows as M or N and its columns as K
// ("K-major"), or with its columns as M or N and its rows as K ("MN-major").
#pragma once

#include <cuda.h>

#include "tgs_common.cuh"

namespace tgs {

constexpr int kBlockCols = 64;          // bf16 columns of an operand block
constexpr int kBlockBytes = 128 * 128;  // a block of 128 rows

// Byte offset of 16-byte unit `unit` (8 columns) of row `row` in a block.
__host__ __device__ __forceinline__ uint32_t unit_offset(uint32_t row, uint32_t unit) {
  return row * 128 + ((unit ^ (row & 7)) << 4);
}

// Shared-memory matrix descriptors, the low word (address / 16, leading
// offset / 16 from bit 16) apart from the high one, which is the same for all:
// stride offset 1024 / 16, descriptor version 1 (bits 46-47), 128-byte swizzle
// (bits 61-63 = 2). Steps of K are additions to the low word.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);

// K-major: 16 columns of K per instruction, 32 bytes along the row.
constexpr uint32_t kStepK = 32 >> 4;
__device__ __forceinline__ uint32_t desc_k(uint32_t block) {
  return ((block & 0x3FFFF) >> 4) | (1u << 16);
}

// MN-major: 16 rows of K per instruction, 2048 bytes; 64 columns of M or N
// per block, the next 64 in the block `lead` bytes on.
constexpr uint32_t kStepMn = 2048 >> 4;
__device__ __forceinline__ uint32_t desc_mn(uint32_t block, uint32_t lead) {
  return ((block & 0x3FFFF) >> 4) | ((lead >> 4) << 16);
}

// Instruction descriptor: fp32 accumulators, bf16 operands, M = 128.
__host__ __device__ constexpr uint32_t tc_idesc(int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
         (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}

// Waits for `phase` of `bar`, two seconds at most. Reading the clock between
// probes paces them: without it, or with a time for the probes to sleep, the
// waits end later (dX of 2,097,152 rows of 64 -> 128 -> 48: 298 and 291 us
// against 245).
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t phase) {
  if (mbar_try_wait(bar, phase)) return true;
  uint64_t start, now;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(start));
  for (uint32_t it = 0; it < kWaitLimit; ++it) {
    if (mbar_try_wait(bar, phase)) return true;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    if (now - start > 2000000000ull) return false;
  }
  return false;
}

// One lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t on;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "elect.sync _|p, 0xffffffff;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(on));
  return on != 0;
}

__device__ __forceinline__ void tc_mma(uint32_t acc, uint32_t a, uint32_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 da, db;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "mov.b64 da, {%1, %5};\n"
      "mov.b64 db, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n"
      "}\n" ::"r"(acc),
      "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate)), "r"(kDescHigh)
      : "memory");
}

// kMost or fewer (`steps`) instructions along K, issued by one lane; the
// whole warp comes here.
template <int kMost>
__device__ __forceinline__ void tc_mma_steps(uint32_t acc, uint32_t a, uint32_t a_step, uint32_t b,
                                             uint32_t b_step, uint32_t idesc, int steps,
                                             bool accumulate) {
  if (elect_one()) {
    if (steps >= kMost) {  // most often: no branch between the instructions
#pragma unroll
      for (int k = 0; k < kMost; ++k)
        tc_mma(acc, a + k * a_step, b + k * b_step, idesc, accumulate || k > 0);
    } else {
#pragma unroll 1
      for (int k = 0; k < steps; ++k)
        tc_mma(acc, a + k * a_step, b + k * b_step, idesc, accumulate || k > 0);
    }
  }
  __syncwarp();
}

// Arrives on `bar` when every matrix instruction issued so far has completed.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  if (elect_one())
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     smem_addr(bar))
                 : "memory");
  __syncwarp();
}

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// A whole warp allocates `cols` columns (a power of two, at least 32).
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_addr(slot)),
               "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
}

// 8 or 16 columns of this warp's 32 lanes: lane l of the quarter holds row l.
// The registers hold the values only after tmem_wait_ld, which is given them
// so that no use of them can move ahead of it.
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]),
        "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]),
        "=f"(v[14]), "=f"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld(float (&v)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]),
                 "+f"(v[7])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]),
                 "+f"(v[7]), "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]),
                 "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// One box of a 2-D tensor map -> shared memory, completion counted on `bar`.
// `col` x the element size is a multiple of 16 bytes.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int col, int row,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(dst),
      "l"(map), "r"(col), "r"(row), "r"(smem_addr(bar))
      : "memory");
}

// Map of a row-major bf16 matrix for boxes of 128 rows x 64 columns in the
// operand layout, zeros outside the matrix. The base is 16-byte aligned and
// the row stride a multiple of 8 elements. Returns a TGS_ status.
int make_row_map(CUtensorMap* map, const void* base, int64_t rows, int cols, int64_t stride);

}  // namespace tgs
