// PTX wrappers for the fifth-generation tensor cores beyond tile_mma.cu's: products of two shared-memory operands,
// operands whose rows run along the contraction (MN-major), 64-row products, and tensor-memory loads and stores of
// the widths that linear attention uses.
#pragma once

#include "common.cuh"

namespace sc {
namespace tc {

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// this thread's shared-memory writes before what the tensor cores read next
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Operands lie in 128-byte swizzle atoms: 8 rows of 128 bytes, the 16-byte piece p of row r at place p ^ (r % 8).
// K-major (a row holds 64 values of the contraction): atoms of 8 rows 1024 bytes apart.
// MN-major (a row holds 64 values of M or N, rows run along the contraction): atoms of 8 rows 1024 bytes apart, the
// next 64 values of M or N `next64` bytes on.
__device__ __forceinline__ uint64_t desc_k(const void* p) {
  return uint64_t((smem_u32(p) & 0x3FFFF) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ uint64_t desc_mn(const void* p, uint32_t next64) {
  return uint64_t((smem_u32(p) & 0x3FFFF) >> 4) | (uint64_t(next64 >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}

// kind::f16 with bfloat16 operands and a float32 accumulator
__host__ __device__ constexpr uint32_t idesc_bf16(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t(a_mn) << 15) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) |
         (uint32_t(m >> 4) << 24);
}

// D (tensor memory) (+)= A B^T, both in shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc))
      : "memory");
}
// the same with A in tensor memory (128 lanes, two values a column)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(acc))
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, e;\n\t}"
      : "=r"(p));
  return p != 0;
}

#define SC_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define SC_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])

__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16 columns of this thread's lane (a warp reads the 32 lanes of its quarter); wait_ld before the registers are used
__device__ __forceinline__ void ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : SC_R8(r, 0), SC_R8(r, 8)
      : "r"(addr));
}
// 16 lanes by 32 columns, as accumulator fragments: thread (g, t) = (lane / 4, lane % 4) gets, for columns 8 j + 2t and
// + 1, row g in r[4j], r[4j + 1] and row g + 8 in r[4j + 2], r[4j + 3]
__device__ __forceinline__ void ld_frag32(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : SC_R8(r, 0), SC_R8(r, 8)
      : "r"(addr));
}
__device__ __forceinline__ void st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), SC_W8(r, 0)
               : "memory");
}
#undef SC_R8
#undef SC_W8

}  // namespace tc
}  // namespace sc
