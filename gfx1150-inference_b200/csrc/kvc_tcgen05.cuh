// tcgen05 building blocks (sm_100a): tensor memory allocation, loads and stores,
// shared-memory matrix descriptors and the 16-bit MMA with fp32 accumulators.
#pragma once

#include <stdint.h>

#include "kvc_device.cuh"

namespace kvc {

// ---- tensor memory ---------------------------------------------------------------
// One warp allocates `cols` columns (a power of two, at least 32); the base address
// lands in shared memory at `dst`.
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst),
               "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// Keeps uses of loaded registers behind the wait for them (no instruction).
template <int N>
__device__ __forceinline__ void tmem_loaded(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
// Order tensor-memory accesses around a synchronisation of threads.
__device__ __forceinline__ void tmem_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tmem_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// 32 lanes x 16 or 32 columns of 32 bits: thread i of the warp has lane i.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// ---- matrix operands ---------------------------------------------------------------
// Descriptor of an unswizzled operand made of 128-byte core matrices (8 rows of 16
// bytes).  `lead` and `stride` are the byte distances between neighbouring core
// matrices: along k and along m/n where k is contiguous in a row of a core matrix; along
// k and along m/n too where m/n is.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(lead >> 4) << 16) |
         (static_cast<uint64_t>(stride >> 4) << 32) | (1ull << 46);
}
// Rows of q, k-major and swizzled: 128-row blocks of kChunk elements (128 bytes where the head
// dim is made of them, else 64) a row, whose 16-byte pieces are permuted by the row number.  A
// copy of 16 bytes a lane then takes whole lines and writes every bank once, where pieces 128
// bytes apart wrote a quarter of them four times (256 rows of 128 dims in the pool's layout took
// an SM 6000 cycles, now one warp 3600).
template <int D>
struct RowBlocks {
  static constexpr int kChunk = D % 64 == 0 ? 64 : 32;          // elements
  static constexpr int kPieces = kChunk / 8;                    // of a row
  static constexpr int kRowsPer = 32 / kPieces;                 // rows that a warp copies at a time
  static constexpr int kBytes = 128 * kChunk * 2;               // of a block
  // Byte offset of piece j of row r of a block.
  static __device__ __forceinline__ uint32_t place(int r, int j) {
    return r * (kChunk * 2) + ((j ^ (kChunk == 64 ? r & 7 : (r >> 1) & 3)) << 4);
  }
  static __device__ __forceinline__ uint64_t desc(uint32_t addr) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) | (1ull << 16) |
           (static_cast<uint64_t>(8 * kChunk * 2 >> 4) << 32) | (1ull << 46) |
           ((kChunk == 64 ? 2ull : 4ull) << 61);
  }
  // What a descriptor grows by for k step k (16 elements).
  static __host__ __device__ constexpr uint64_t step(int k) {
    return static_cast<uint64_t>((k * 16 / kChunk * kBytes + k * 16 % kChunk * 2) >> 4);
  }
};
// Instruction descriptor: A and B of one 16-bit type, fp32 accumulators.
template <typename T>
__host__ __device__ constexpr uint32_t mma_desc(int m, int n, bool b_mn_major);
template <>
__host__ __device__ constexpr uint32_t mma_desc<__half>(int m, int n, bool b_mn_major) {
  return (1u << 4) | (b_mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
template <>
__host__ __device__ constexpr uint32_t mma_desc<__nv_bfloat16>(int m, int n, bool b_mn_major) {
  return mma_desc<__half>(m, n, b_mn_major) | (1u << 7) | (1u << 10);
}
// D[tmem] (+)= A[smem] B[smem], one k step of 16.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
      : "memory");
}
// The mbarrier arrives when every MMA this thread issued before is done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
      : "memory");
}

}  // namespace kvc
