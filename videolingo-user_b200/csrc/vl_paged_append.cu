// Rotary embedding of q and k with the append of k and v to a paged KV cache.
//
// Token t of sequence b sits at position p = kv_len[b] - (q_start[b+1] - t);
// its k and v rows go to row p % page of page page_table[b][p / page].  Pair
// d < rot/2 of a head turns by the angle p * scale * base^(-2d/rot):
//   x1' = x1 cos - x2 sin,  x2' = x2 cos + x1 sin
// over (d, d + rot/2), or over (2d, 2d + 1) when interleaved.
//
// The op moves 2 * (n_q + 2 n_kv) * head_dim elements per token and computes
// next to nothing, so it is bound by HBM, or for a decode step by the
// latency of one round trip (q_start -> page id -> store).
//
// Layout: a warp takes heads of one token, a lane one 16-byte vector of a
// head; every access of a warp is one contiguous 512 bytes.  A rotate-half
// lane gets the other half of its pairs from the lane half a rotation away
// by shuffle, so a vector is loaded once and the same code serves every
// rotary_dim; interleaved pairs lie within a lane.  A lane's vector index is
// the same in every head, so its cosines and sines are evaluated once per
// token.  Vector loads are requested before the angles are evaluated.
#include <cmath>

#include "vl_common.cuh"
#include "vl_kernels.h"
#include "vl_paged.cuh"
#include "vl_rope_math.cuh"

namespace vl {
namespace {

constexpr int kAppendWarps = 4;
constexpr int kAppendAhead = 6;   // head rows a lane holds in flight

// wpt warps share a token's heads (1, 2 or 4, so that few tokens still
// spread over the SMs).
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kAppendWarps * 32)
    paged_append_kernel(const __grid_constant__ PagedAppendArgs a,
                        const __grid_constant__ InvFreq freq, int wpt) {
  using S = Storage<T>;
  constexpr int E = S::kVec;
  __shared__ float2 cs_all[kAppendWarps][kMaxHalfRot];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t wid = static_cast<int64_t>(blockIdx.x) * kAppendWarps + warp;
  const int64_t t = wid / wpt;
  const int part = static_cast<int>(wid % wpt);
  if (t >= a.tokens) return;

  const int nv = a.head_dim / E;            // vectors of a head, <= 32
  const int hpw = 32 / nv;                  // heads of a warp row
  const int v = lane % nv, hl = lane / nv;
  const bool lane_on = hl < hpw;
  const int heads = a.n_q_heads + 2 * a.n_kv_heads;
  const int kv0 = a.n_q_heads, v0 = a.n_q_heads + a.n_kv_heads;
  const int half_vecs = a.rotary_dim / 2 / E;   // rotate-half: vectors of a half
  const bool rotates = v * E < a.rotary_dim;

  auto source = [&](int h) -> const T* {
    if (h < kv0)
      return static_cast<const T*>(a.q) + t * a.q_row_stride + static_cast<int64_t>(h) * a.head_dim;
    if (h < v0)
      return static_cast<const T*>(a.k) + t * a.k_row_stride +
             static_cast<int64_t>(h - kv0) * a.head_dim;
    return static_cast<const T*>(a.v) + t * a.v_row_stride +
           static_cast<int64_t>(h - v0) * a.head_dim;
  };
  const int step = hpw * wpt;
  uint4 x[kAppendAhead];
  auto load = [&](int h0) {
#pragma unroll
    for (int i = 0; i < kAppendAhead; ++i) {
      const int h = h0 + i * step + hl;
      if (lane_on && h < heads) x[i] = ld_vec(source(h) + v * E);
    }
  };
  // the rows are readable whether or not a sequence holds them
  load(part * hpw);

  const int b = find_sequence(a.q_start, a.batch, t, lane);
  const int64_t q0 = a.q_start[b], q1 = a.q_start[b + 1];
  if (t < q0 || t >= q1) return;            // behind the last sequence
  const int64_t pos = static_cast<int64_t>(a.kv_len[b]) - (q1 - t);
  const int shift = ilog2(a.page_size);
  const int64_t page_at = pos >> shift;
  int64_t page = -1;
  if (pos >= 0 && page_at < a.max_pages) page = a.page_table[b * a.table_stride + page_at];
  const bool cached = page >= 0 && page < a.num_pages;
  if (!cached && part == 0 && lane == 0 && a.status) atomicOr(a.status, VL_STATUS_BAD_PAGE);
  const int64_t at = page * a.page_stride +
                     (pos & (a.page_size - 1)) * static_cast<int64_t>(a.n_kv_heads) * a.head_dim;

  float2* cs = cs_all[warp];
  const double angle = static_cast<double>(pos) * a.position_scale;
  for (int d = lane; d < a.rotary_dim / 2; d += 32) cs[d] = rope_cos_sin(angle * freq.v[d]);
  __syncwarp();
  float c[E], s[E];
  if (kInterleaved) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float2 p = rotates ? cs[v * (E / 2) + e / 2] : make_float2(1.0f, 0.0f);
      c[e] = p.x;
      s[e] = (e & 1) ? p.y : -p.y;          // x1' = x1 c - x2 s, x2' = x2 c + x1 s
    }
  } else {
    const bool second = v >= half_vecs;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float2 p = rotates ? cs[(second ? v - half_vecs : v) * E + e] : make_float2(1.0f, 0.0f);
      c[e] = p.x;
      s[e] = second ? p.y : -p.y;
    }
  }
  const int partner = kInterleaved || !rotates ? lane
                      : (v >= half_vecs ? lane - half_vecs : lane + half_vecs);

  for (int h0 = part * hpw; h0 < heads; h0 += kAppendAhead * step) {
    if (h0 != part * hpw) load(h0);
#pragma unroll
    for (int i = 0; i < kAppendAhead; ++i) {
      const int hw = h0 + i * step;         // warp-uniform
      if (hw >= heads) break;
      const int h = hw + hl;
      uint4 o = x[i];
      if (!kInterleaved) {
        o.x = __shfl_sync(0xffffffffu, x[i].x, partner);
        o.y = __shfl_sync(0xffffffffu, x[i].y, partner);
        o.z = __shfl_sync(0xffffffffu, x[i].z, partner);
        o.w = __shfl_sync(0xffffffffu, x[i].w, partner);
      }
      if (!lane_on || h >= heads) continue;
      uint4 y = x[i];
      if (h < v0 && rotates) {
        float f[E], g[E], r[E];
        S::unpack(x[i], f);
        S::unpack(o, g);
#pragma unroll
        for (int e = 0; e < E; ++e) r[e] = f[e] * c[e] + (kInterleaved ? g[e ^ 1] : g[e]) * s[e];
        y = S::pack(r);
      }
      T* dst;
      if (h < kv0) {
        dst = static_cast<T*>(a.q_out) + t * a.q_out_row_stride +
              static_cast<int64_t>(h) * a.head_dim;
      } else {
        if (!cached) continue;
        dst = h < v0 ? static_cast<T*>(a.k_cache) + at + static_cast<int64_t>(h - kv0) * a.head_dim
                     : static_cast<T*>(a.v_cache) + at + static_cast<int64_t>(h - v0) * a.head_dim;
      }
      st_vec(dst + v * E, y);
    }
  }
}

// Any head_dim, rotary_dim, stride or alignment: a block per token, one
// element pair per thread.
template <typename T>
__global__ void __launch_bounds__(128)
    paged_append_scalar_kernel(const __grid_constant__ PagedAppendArgs a,
                               const __grid_constant__ InvFreq freq) {
  using S = Storage<T>;
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 31;
  const int b = find_sequence(a.q_start, a.batch, t, lane);
  const int64_t q0 = a.q_start[b], q1 = a.q_start[b + 1];
  if (t < q0 || t >= q1) return;
  const int64_t pos = static_cast<int64_t>(a.kv_len[b]) - (q1 - t);
  const int64_t page_at = pos >> ilog2(a.page_size);
  int64_t page = -1;
  if (pos >= 0 && page_at < a.max_pages) page = a.page_table[b * a.table_stride + page_at];
  const bool cached = page >= 0 && page < a.num_pages;
  if (!cached && threadIdx.x == 0 && a.status) atomicOr(a.status, VL_STATUS_BAD_PAGE);
  const int64_t at = page * a.page_stride +
                     (pos & (a.page_size - 1)) * static_cast<int64_t>(a.n_kv_heads) * a.head_dim;
  const int half = a.rotary_dim / 2, rest = a.head_dim - a.rotary_dim;
  const int per_head = half + rest;         // pairs, then single elements
  const int heads = a.n_q_heads + 2 * a.n_kv_heads;
  const int kv0 = a.n_q_heads, v0 = kv0 + a.n_kv_heads;
  for (int i = threadIdx.x; i < heads * per_head; i += blockDim.x) {
    const int h = i / per_head, j = i - h * per_head;
    const T* src;
    T* dst;
    if (h < kv0) {
      src = static_cast<const T*>(a.q) + t * a.q_row_stride + static_cast<int64_t>(h) * a.head_dim;
      dst = static_cast<T*>(a.q_out) + t * a.q_out_row_stride +
            static_cast<int64_t>(h) * a.head_dim;
    } else {
      if (!cached) continue;
      const int64_t hk = h < v0 ? h - kv0 : h - v0;
      src = (h < v0 ? static_cast<const T*>(a.k) + t * a.k_row_stride
                    : static_cast<const T*>(a.v) + t * a.v_row_stride) + hk * a.head_dim;
      dst = (h < v0 ? static_cast<T*>(a.k_cache) : static_cast<T*>(a.v_cache)) + at +
            hk * a.head_dim;
    }
    if (j >= half) {
      const int d = a.rotary_dim + j - half;
      dst[d] = src[d];
      continue;
    }
    const int d1 = a.interleaved ? 2 * j : j, d2 = a.interleaved ? 2 * j + 1 : j + half;
    const T e1 = src[d1], e2 = src[d2];
    if (h >= v0) {
      dst[d1] = e1;
      dst[d2] = e2;
      continue;
    }
    const float2 cs = rope_cos_sin(static_cast<double>(pos) * a.position_scale * freq.v[j]);
    const float x1 = S::to_float(e1), x2 = S::to_float(e2);
    dst[d1] = S::from_float(x1 * cs.x - x2 * cs.y);
    dst[d2] = S::from_float(x2 * cs.x + x1 * cs.y);
  }
}

template <typename T>
cudaError_t append_typed(const PagedAppendArgs& a, cudaStream_t stream) {
  constexpr int E = Storage<T>::kVec;
  const InvFreq freq = make_inv_freq(a.base, a.rotary_dim);
  const bool rot_vec = a.interleaved ? a.rotary_dim % E == 0 : (a.rotary_dim / 2) % E == 0;
  const bool vec = a.head_dim % E == 0 && a.head_dim / E <= 32 && rot_vec &&
                   a.page_stride % E == 0 && a.k_row_stride % E == 0 && a.v_row_stride % E == 0 &&
                   aligned16(a.k) && aligned16(a.v) && aligned16(a.k_cache) &&
                   aligned16(a.v_cache) &&
                   (a.n_q_heads == 0 || (aligned16(a.q) && aligned16(a.q_out) &&
                                         a.q_row_stride % E == 0 && a.q_out_row_stride % E == 0));
  if (!vec) {
    paged_append_scalar_kernel<T><<<static_cast<unsigned>(a.tokens), 128, 0, stream>>>(a, freq);
    return cudaGetLastError();
  }
  const int64_t sms = sm_count();
  const int wpt = a.tokens <= 4 * sms ? 4 : (a.tokens <= 8 * sms ? 2 : 1);
  const int64_t blocks = (a.tokens * wpt + kAppendWarps - 1) / kAppendWarps;
  if (a.interleaved)
    paged_append_kernel<T, true>
        <<<static_cast<unsigned>(blocks), kAppendWarps * 32, 0, stream>>>(a, freq, wpt);
  else
    paged_append_kernel<T, false>
        <<<static_cast<unsigned>(blocks), kAppendWarps * 32, 0, stream>>>(a, freq, wpt);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendArgs& a, int dtype, cudaStream_t stream) {
  if (a.tokens == 0) return cudaSuccess;
  switch (dtype) {
    case kDtypeF32: return append_typed<float>(a, stream);
    case kDtypeF16: return append_typed<__half>(a, stream);
    default: return append_typed<__nv_bfloat16>(a, stream);
  }
}

}  // namespace vl
