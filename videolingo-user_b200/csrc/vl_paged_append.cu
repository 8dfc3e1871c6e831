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
// Layout: a block takes a few tokens.  Its first threads look the tokens'
// places up, then all of them evaluate the tokens' cosines and sines (once
// per token, in shared memory) while the first vectors are on their way, and
// then move 16-byte vectors: a task is the two vectors of a head that turn
// together (one, when interleaved), or one that is only copied.
//
// 16 x 383 tokens, 16 / 4 heads of 128, bf16 (75 MB): 18.3 us, 0.63 of the
// measured copy rate; issue slots are 0.57 busy, the rest is what the short
// blocks wait for (lookup, sincosf, first vectors).  16 x 1: 3.1 us.
#include <cmath>

#include "vl_common.cuh"
#include "vl_kernels.h"
#include "vl_paged.cuh"
#include "vl_rope_math.cuh"

namespace vl {
namespace {

constexpr int kAppendThreads = 256;
// Tasks of a thread in flight: a task that turns two vectors holds twice the
// registers.  With three of those five blocks fit on an SM (16 x 383 tokens:
// 18.3 us, with four and four blocks 0.6 more).  Interleaved ones fit six with four
// as they come (37 ragged sequences: 53.2 us, 62.8 with three; held to six
// blocks 55.1).
constexpr int append_ahead(bool interleaved) { return interleaved ? 4 : 3; }
constexpr int kAppendTokens = 4;  // of a block, at most

// n / d for n, d < 2^16 by the factor ceil(2^32 / d).
struct Divisor {
  uint32_t d, factor;
};
__device__ __forceinline__ int quotient(int n, const Divisor& v) {
  return v.d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), v.factor));
}

struct AppendTasks {
  int turns;        // of a token: (q and k heads) * vectors (pairs of vectors) that turn
  int tails;        // (q and k heads) * vectors behind rotary_dim
  Divisor token;    // turns + tails + v heads * vectors
  Divisor turn;     // turning tasks of a head
  Divisor tail;
  Divisor whole;    // vectors of a head
};

template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads, kInterleaved ? 0 : 5)
    paged_append_kernel(const __grid_constant__ PagedAppendArgs a,
                        const __grid_constant__ InvFreq freq,
                        const __grid_constant__ AppendTasks tasks, int block_tokens) {
  using S = Storage<T>;
  constexpr int E = S::kVec;
  constexpr int G = append_ahead(kInterleaved);
  constexpr int kPairs = kInterleaved ? E / 2 : E;   // of a task
  __shared__ __align__(16) float2 cs[kAppendTokens * kMaxHalfRot];
  __shared__ int64_t s_at[kAppendTokens];   // the cache row's offset, -1: not cached, -2: no token
  __shared__ int s_pos[kAppendTokens];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * block_tokens;
  const int nt = static_cast<int>(min(static_cast<int64_t>(block_tokens), a.tokens - t0));
  const int half = a.rotary_dim / 2;
  const int kv0 = a.n_q_heads;
  const int count = nt * static_cast<int>(tasks.token.d);

  struct Task {
    int token, head, vec;   // head: q, then k, then v heads
    bool turns;
  };
  auto task_of = [&](int n) {
    Task k;
    k.token = quotient(n, tasks.token);
    int m = n - k.token * static_cast<int>(tasks.token.d);
    k.turns = m < tasks.turns;
    if (k.turns) {
      k.head = quotient(m, tasks.turn);
      k.vec = m - k.head * static_cast<int>(tasks.turn.d);
    } else if ((m -= tasks.turns) < tasks.tails) {
      k.head = quotient(m, tasks.tail);
      k.vec = a.rotary_dim / E + m - k.head * static_cast<int>(tasks.tail.d);
    } else {
      m -= tasks.tails;
      const int h = quotient(m, tasks.whole);
      k.head = kv0 + a.n_kv_heads + h;
      k.vec = m - h * static_cast<int>(tasks.whole.d);
    }
    return k;
  };
  auto source = [&](const Task& k) {
    const int64_t t = t0 + k.token;
    const T* row;
    int h = k.head;
    if (h < kv0) {
      row = static_cast<const T*>(a.q) + t * a.q_row_stride;
    } else if ((h -= kv0) < a.n_kv_heads) {
      row = static_cast<const T*>(a.k) + t * a.k_row_stride;
    } else {
      h -= a.n_kv_heads;
      row = static_cast<const T*>(a.v) + t * a.v_row_stride;
    }
    return row + static_cast<int64_t>(h) * a.head_dim + k.vec * E;
  };
  uint4 x1[G], x2[G];
  auto load = [&](int n0) {                 // readable whether or not a sequence holds the token
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int n = n0 + g * kAppendThreads;
      if (n < count) {
        const Task k = task_of(n);
        const T* src = source(k);
        x1[g] = ld_vec(src);
        if (!kInterleaved && k.turns) x2[g] = ld_vec(src + half);
      }
    }
  };
  load(tid);

  if (warp < nt) {                          // a token's place
    const int64_t t = t0 + warp;
    const int b = find_sequence(a.q_start, a.batch, t, lane);
    const int64_t q0 = a.q_start[b], q1 = a.q_start[b + 1];
    const int64_t pos = static_cast<int64_t>(a.kv_len[b]) - (q1 - t);
    int64_t at = -2;
    if (t >= q0 && t < q1) {
      const int64_t page_at = pos >> ilog2(a.page_size);
      int64_t page = -1;
      if (pos >= 0 && page_at < a.max_pages) page = a.page_table[b * a.table_stride + page_at];
      at = -1;
      if (page >= 0 && page < a.num_pages)
        at = page * a.page_stride +
             (pos & (a.page_size - 1)) * static_cast<int64_t>(a.n_kv_heads) * a.head_dim;
      else if (lane == 0 && a.status)
        atomicOr(a.status, VL_STATUS_BAD_PAGE);
    }
    if (lane == 0) {
      s_at[warp] = at;
      s_pos[warp] = static_cast<int>(pos);
    }
  }
  // The frequencies are a kernel parameter: read through a generic address,
  // as constants they would be fetched one lane at a time.
  const double* freqs = freq.v;
  asm volatile("" : "+l"(freqs));
  const int my_d = tid % (half > 0 ? half : 1);
  const double my_f = tid < half * nt ? freqs[my_d] : 0.0;
  __syncthreads();
  for (int i = tid; i < nt * half; i += kAppendThreads) {
    const int t = i / half, d = i - t * half;
    // pair e of vector j at [e][j]: the lanes of a warp read neighbours
    cs[t * kMaxHalfRot + d % kPairs * (half / kPairs) + d / kPairs] =
        rope_cos_sin(static_cast<double>(s_pos[t]) * a.position_scale * (i == tid ? my_f : freqs[d]));
  }
  __syncthreads();

  for (int n0 = tid; n0 < count; n0 += G * kAppendThreads) {
    if (n0 != tid) load(n0);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int n = n0 + g * kAppendThreads;
      if (n >= count) break;
      const Task k = task_of(n);
      const int64_t at = s_at[k.token];
      if (at == -2 || (at == -1 && k.head >= kv0)) continue;
      T* dst;
      int h = k.head;
      if (h < kv0)
        dst = static_cast<T*>(a.q_out) + (t0 + k.token) * a.q_out_row_stride;
      else if ((h -= kv0) < a.n_kv_heads)
        dst = static_cast<T*>(a.k_cache) + at;
      else {
        h -= a.n_kv_heads;
        dst = static_cast<T*>(a.v_cache) + at;
      }
      dst += static_cast<int64_t>(h) * a.head_dim + k.vec * E;
      if (!k.turns) {
        st_vec(dst, x1[g]);
        continue;
      }
      float p[E], y[E];
      S::unpack(x1[g], p);
      if (kInterleaved) {
        const float2* cv = cs + k.token * kMaxHalfRot + k.vec;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 w = cv[e / 2 * (half / kPairs)];
          y[e] = p[e] * w.x - p[e + 1] * w.y;
          y[e + 1] = p[e + 1] * w.x + p[e] * w.y;
        }
        st_vec(dst, S::pack(y));
      } else {
        float r[E], z[E];
        S::unpack(x2[g], r);
        const float2* cv = cs + k.token * kMaxHalfRot + k.vec;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 w = cv[e * (half / kPairs)];
          y[e] = p[e] * w.x - r[e] * w.y;
          z[e] = r[e] * w.x + p[e] * w.y;
        }
        st_vec(dst, S::pack(y));
        st_vec(dst + half, S::pack(z));
      }
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

// base^(-2d / rotary_dim), every eighth and the seven between by pow, the
// others as products of the two: 64 calls of pow cost 0.6 us more of a call's
// host time (6.7 -> 6.1), and a product is within 2 steps of 2^-53 more, 2e-10
// rad at position 2^20.
InvFreq append_inv_freq(double base, int rotary_dim) {
  InvFreq f{};
  const int half = rotary_dim / 2;
  double step[8];
  for (int j = 0; j < 8 && j < half; ++j)
    step[j] = 1.0 / std::pow(base, static_cast<double>(2 * j) / rotary_dim);
  for (int d = 0; d < half && d < kMaxHalfRot; d += 8) {
    const double at = 1.0 / std::pow(base, static_cast<double>(2 * d) / rotary_dim);
    for (int j = 0; j < 8 && d + j < half; ++j) f.v[d + j] = at * step[j];
  }
  return f;
}

template <typename T>
cudaError_t append_typed(const PagedAppendArgs& a, cudaStream_t stream) {
  constexpr int E = Storage<T>::kVec;
  const InvFreq freq = append_inv_freq(a.base, a.rotary_dim);
  const bool rot_vec = a.interleaved ? a.rotary_dim % E == 0 : (a.rotary_dim / 2) % E == 0;
  // (the task numbers of a block stay below 2^16)
  const bool vec = a.head_dim % E == 0 && rot_vec &&
                   (a.n_q_heads + 2 * a.n_kv_heads) * (a.head_dim / E) <= 16384 &&
                   a.page_stride % E == 0 && a.k_row_stride % E == 0 && a.v_row_stride % E == 0 &&
                   aligned16(a.k) && aligned16(a.v) && aligned16(a.k_cache) &&
                   aligned16(a.v_cache) &&
                   (a.n_q_heads == 0 || (aligned16(a.q) && aligned16(a.q_out) &&
                                         a.q_row_stride % E == 0 && a.q_out_row_stride % E == 0));
  if (!vec) {
    paged_append_scalar_kernel<T><<<static_cast<unsigned>(a.tokens), 128, 0, stream>>>(a, freq);
    return cudaGetLastError();
  }
  const int nv = a.head_dim / E, qk = a.n_q_heads + a.n_kv_heads;
  const int turn = a.interleaved ? a.rotary_dim / E : a.rotary_dim / 2 / E;
  const int tail = nv - a.rotary_dim / E;
  auto divisor = [](int d) {
    const uint32_t u = d > 0 ? d : 1;
    return Divisor{u, static_cast<uint32_t>(((uint64_t(1) << 32) + u - 1) / u)};
  };
  AppendTasks tasks;
  tasks.turns = qk * turn;
  tasks.tails = qk * tail;
  tasks.token = divisor(tasks.turns + tasks.tails + a.n_kv_heads * nv);
  tasks.turn = divisor(turn);
  tasks.tail = divisor(tail);
  tasks.whole = divisor(nv);
  // tokens of a block: enough for every thread to have its tasks in flight,
  // but one while there are few blocks
  int block_tokens =
      append_ahead(a.interleaved) * kAppendThreads / static_cast<int>(tasks.token.d);
  if (block_tokens > kAppendTokens) block_tokens = kAppendTokens;
  if (block_tokens < 1 || a.tokens <= 2 * sm_count()) block_tokens = 1;
  const int64_t blocks = (a.tokens + block_tokens - 1) / block_tokens;
  auto kernel = a.interleaved ? paged_append_kernel<T, true> : paged_append_kernel<T, false>;
  kernel<<<static_cast<unsigned>(blocks), kAppendThreads, 0, stream>>>(a, freq, tasks,
                                                                       block_tokens);
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
