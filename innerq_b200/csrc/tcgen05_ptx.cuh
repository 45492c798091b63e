// PTX wrappers for the fifth-generation tensor cores: tensor memory, matrix
// descriptors, tcgen05 instructions, tiled TMA loads (no multicast).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "async_ptx.cuh"

namespace innerq {

// ------------------------------------------------------- tensor memory ---
// 512 columns of 128 lanes of 32 bits; an address is lane << 16 | column
__device__ __forceinline__ void tmem_alloc(uint32_t* out, int columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(out)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, int columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(addr), "r"(columns) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// 32 consecutive columns of this warp's 32 lanes, one lane per thread
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const float* r) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(r);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
      "%31,%32};\n" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]),
      "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]),
      "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(addr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}

// --------------------------------------------------------- descriptors ---
// Shared-memory operand in 128-byte-swizzled atoms of 8 rows x 128 bytes.
// K-major (rows along M / N, K contiguous): sbo = bytes between 8-row groups.
// MN-major (rows along K, M / N contiguous): lbo = bytes between 128-byte
// column blocks, sbo = bytes between 8-row groups.  The descriptor's low word
// holds address and lbo in units of 16 bytes (adding to it moves the operand),
// the high word is a constant.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo) { return (addr >> 4 & 0x3fff) | (lbo >> 4) << 16; }
__host__ __device__ constexpr uint32_t desc_hi(uint32_t sbo) { return sbo >> 4 | 1u << 14 | 2u << 29; }
// kind::f16 instruction: fp32 accumulator, A and B both f16 (0) or bf16 (1),
// A K-major, B K-major or MN-major
__host__ __device__ constexpr uint32_t mma_idesc(int M, int N, int dtype, int b_mn_major) {
  return 1u << 4 | (uint32_t)dtype << 7 | (uint32_t)dtype << 10 | (uint32_t)b_mn_major << 16 | (uint32_t)(N >> 3) << 17 |
         (uint32_t)(M >> 4) << 24;
}

// One lane of a converged warp.  The warp that issues MMAs stays converged and
// its instructions carry this predicate: operands that are uniform over the
// warp then live in uniform registers, where tcgen05 wants them.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r;
}
// D (tensor memory) = A B (+ D)
template <uint32_t AHI, uint32_t BHI>
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 a, b;\n setp.ne.u32 p, %5, 0;\n setp.ne.u32 q, %4, 0;\n"
      " mov.b64 a, {%1, %6};\n mov.b64 b, {%2, %7};\n"
      " @p tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, q;\n}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(acc), "r"(leader), "n"(AHI), "n"(BHI)
      : "memory");
}
template <uint32_t BHI>
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 b;\n setp.ne.u32 p, %5, 0;\n setp.ne.u32 q, %4, 0;\n"
      " mov.b64 b, {%2, %6};\n"
      " @p tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, q;\n}\n" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(idesc), "r"(acc), "r"(leader), "n"(BHI)
      : "memory");
}
// the barrier gets one arrival when every MMA the leader issued is complete
__device__ __forceinline__ void mma_commit(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %1, 0;\n"
      " @p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}

// ----------------------------------------------------------------- TMA ---
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];\n" ::"l"(map) : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];\n" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// -------------------------------------------------- taking over blocks ---
// Ask for a block of this grid that has not been launched yet: 16 bytes at
// `answer`, completing `bar`.  After a "no" it must not be asked again.
__device__ __forceinline__ void next_block_ask(void* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
// its blockIdx.x, or -1: there is none
__device__ __forceinline__ int next_block_get(const void* answer) {
  int x;
  asm volatile(
      "{\n .reg .pred p;\n .reg .b128 h;\n .reg .b32 y, z, w;\n ld.shared.b128 h, [%1];\n mov.b32 %0, -1;\n"
      " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
      " @p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, y, z, w}, h;\n}\n"
      : "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return x;
}

}  // namespace innerq
