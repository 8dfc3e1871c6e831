// mbarrier, TMA and tensor-map helpers of the paged-attention kernels.
#pragma once

#include <cuda.h>

#include "vl_common.cuh"

namespace vl {

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbarrier_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count)
               : "memory");
}
__device__ __forceinline__ void mbarrier_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbarrier_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ bool mbarrier_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbarrier_test(uint64_t* bar, uint32_t parity) {
  return mbarrier_test(smem_addr(bar), parity);
}
constexpr uint32_t kWaitPolls = 1u << 22;   // try_wait suspends: some seconds

// One lane of a converged warp, to issue MMAs or TMA copies: these take their
// operands from uniform registers, and issued lane by lane, or in a loop that
// makes its descriptors as it goes, they cost about 200 cycles each; unrolled
// behind an elected lane, what the hardware needs (64 for a 128 x 128 x 16
// MMA).
__device__ __forceinline__ bool elect_lane() {
  uint32_t on;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(on));
  return on != 0;
}
// Waits for the phase of the given parity, a few seconds at most: false then.
__device__ __forceinline__ bool mbarrier_wait(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < kWaitPolls; ++i)
    if (mbarrier_test(bar, parity)) return true;
  return false;
}

// A run of 16-byte units into shared memory (both ends on 16-byte boundaries).
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(smem_addr(bar))
      : "memory");
}

// A box of a 4-D tensor map ([pages][page rows][kv heads][head dims]).
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int dim,
                                            int head, int row, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(dim), "r"(head), "r"(row), "r"(page),
      "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int dim,
                                            int head, int row, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(dim), "r"(head), "r"(row), "r"(smem_addr(bar))
      : "memory");
}

// Tensor map of a 16-bit cache, boxes of 64 head dims x 1 head x box_rows
// rows of one page in the 128-byte swizzle.  False if the driver refuses.
bool encode_cache_map(CUtensorMap* map, const void* cache, bool bf16, int head_dim,
                      int n_kv_heads, int page_size, int64_t num_pages, int64_t page_stride,
                      int box_rows);
// Tensor map of packed 16-bit q rows, boxes of 64 head dims x box_heads heads x
// box_tokens rows in the 128-byte swizzle.
bool encode_rows_map(CUtensorMap* map, const void* rows, bool bf16, int head_dim, int n_heads,
                     int64_t tokens, int64_t row_stride, int box_heads, int box_tokens);

}  // namespace vl
