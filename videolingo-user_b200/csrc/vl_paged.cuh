// Shared by the paged-cache and beam-search kernels: which sequence a packed
// row belongs to, whether a sequence's device-side lengths are usable, and
// arithmetic that fp32 code has no operators for.
#pragma once

#include "vl_common.cuh"
#include "vl_kernels.h"

namespace vl {

__device__ __forceinline__ int ilog2(int pow2) { return 31 - __clz(pow2); }

// 64-bit division, at the price of a 32-bit one where that will do.
__device__ __forceinline__ int64_t divide(int64_t x, int64_t y) {
  if (((x | y) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
  return x / y;
}

constexpr float kLog2e = 1.4426950408889634f;

// Two values as 16-bit ones of a type, the first in the low half.
__device__ __forceinline__ uint32_t pack16(float lo, float hi, __nv_bfloat16) {
  return pack_bf16x2(lo, hi);
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, __half) {
  return pack_f16x2(lo, hi);
}

// The exponential unit's 2^x (relative error below 2^-22).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two floats in one 64-bit register, for the packed adds and multiply-adds
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ uint64_t pair_of(uint32_t a, uint32_t b) {
  uint64_t y;
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "r"(a), "r"(b));
  return y;
}
__device__ __forceinline__ float2 halves_of(uint64_t x) {
  float2 y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(x));
  return y;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(a), "l"(b), "l"(c));
  return y;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t y;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(y) : "l"(a), "l"(b));
  return y;
}

// The largest b in [0, batch) with q_start[b] <= row, or 0: the sequence of
// a packed row if any holds it.  Called by a whole warp; 32 probes a round.
__device__ __forceinline__ int find_sequence(const int32_t* __restrict__ q_start, int batch,
                                             int64_t row, int lane) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int p = lo + (lane + 1) * step;
    const bool at_or_before = p < hi && static_cast<int64_t>(q_start[p]) <= row;
    const int n = __popc(__ballot_sync(0xffffffffu, at_or_before));
    lo += n * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// A sequence of a ragged batch as the attention kernels see it.
struct SeqView {
  int start;   // first packed row
  int rows;    // new tokens (0: nothing to do)
  int len;     // cached positions, new tokens included (0: zero output rows)
  bool bad;    // lengths out of range
};

__device__ __forceinline__ SeqView sequence_view(const PagedAttnArgs& a, int b, int page_shift) {
  SeqView s;
  const int q0 = a.q_start[b], q1 = a.q_start[b + 1];
  const int len = a.kv_len[b];
  s.start = q0;
  s.rows = q1 - q0;
  s.len = len;
  s.bad = false;
  if (q0 < 0 || q1 < q0 || static_cast<int64_t>(q1) > a.tokens) {
    s.start = 0;   // no rows that could be told to be this sequence's
    s.rows = 0;
    s.len = 0;
    s.bad = true;
  } else if (len < 0 || static_cast<int64_t>(len) > (static_cast<int64_t>(a.max_pages) << page_shift) ||
             s.rows > a.max_q_len) {
    s.len = 0;
    s.bad = true;
  }
  return s;
}

}  // namespace vl
