// Beam search for sm_100a: the selection of the best continuations over
// beams and vocabulary, and the reordering of paged caches after it.
//
// Selection.  A live beam b offers token v at s_b + l_bv - lse_b with
// lse_b = log sum_v exp(l_bv); the entry keeps the `beams` largest values,
// ties to the lower b * vocab + v.  Within a row the order is that of the
// logits, so the logits are read once: CTAs stream pieces of rows and keep
// the maximum, the sum of exponentials about it and the `beams` largest
// logits; a second launch merges the pieces of the rows and the rows of an
// entry.  It is bound by the read of the logits (about eight instructions an
// element keep up with it) and by what a piece costs by itself, or for one
// entry by two launches' latency: 64 x 5 f32 rows of 51865, some finished
// (53 MB), 20.9 us, 64 x 5 bf16 rows of 59264 (38 MB) 24.6, 1 x 4 of them 10.4.
//   * The K-th largest of the lanes' maxima of the first round bounds the K-th
//     largest value from below and lets few values through (a few dozen of
//     50,000, as what gets through raises the bound again): these go to a
//     heap in shared memory, which is sorted at the end.  What does not fit
//     (rows in ascending order, rows of equal values) goes to a list per warp,
//     one entry a lane, best first, whose last entry then is the bound;
//     values come in index order, so equal ones keep it.  Inserting into a
//     list takes a warp some 700 cycles, a place on the heap a lane 100.
//   * Lists are merged pairwise as bitonic sequences, five exchanges each.
//   * exp is taken of l - m, m the lane's maximum at its last rescaling, summed
//     in fp32 over a round (chains of 16 values) and in fp64 above that; values
//     are compared in fp64.  Two beams are told apart to 1e-5, the error of
//     their lse at any vocab: 20 * 2^-24 by a round's additions, 2^-22 by ex2,
//     and for its argument 2.5 * 2^-24 times the distance from m, which is 17
//     where 2^24 values share a row's mass, and the last two once more for a
//     lane's three rescalings that weigh (kSelLag) and the joins of lanes and
//     pieces: 6e-6 together.  Within a row the order is exact.
//
// Reordering.  See vl_paged_beam_reorder in vl_api.h for the rule.  Every
// CTA of an entry works the small plan out for itself (a bitmap of the
// entry's range in shared memory), so one launch does tables and copies and
// nothing waits for another CTA.  Bound by the copies: 32 x 5 rows over 28
// layers (119 MB moved) 23.6 us, 0.77 of the measured copy rate; 4 x 4 rows
// 6.0 us, the plan's chain of look-ups.
#include <atomic>
#include <cmath>

#include "vl_common.cuh"
#include "vl_kernels.h"
#include "vl_paged.cuh"
#include "vl_tma.cuh"

namespace vl {
namespace {

constexpr float kNegInf = -INFINITY;
constexpr int kNoIndex = 0x7fffffff;

// ---------------------------------------------------------------------------
// sorted lists, one entry per lane, best first
// ---------------------------------------------------------------------------
template <typename V>
__device__ __forceinline__ bool better(V v, int i, V w, int j) {
  return v > w || (v == w && i < j);
}

// The best 32 of two sorted lists of 32, sorted.
template <typename V>
__device__ __forceinline__ void merge_lists(V& v, int& i, V w, int j, int lane) {
  const V wr = __shfl_sync(0xffffffffu, w, 31 - lane);
  const int jr = __shfl_sync(0xffffffffu, j, 31 - lane);
  if (better(wr, jr, v, i)) {
    v = wr;
    i = jr;
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const V ov = __shfl_xor_sync(0xffffffffu, v, s);
    const int oi = __shfl_xor_sync(0xffffffffu, i, s);
    const bool first = (lane & s) == 0;
    if (better(ov, oi, v, i) == first) {
      v = ov;
      i = oi;
    }
  }
}

// 32 entries in any order into a list.
template <typename V>
__device__ __forceinline__ void sort_list(V& v, int& i, int lane) {
#pragma unroll
  for (int n = 2; n <= 32; n <<= 1) {      // runs of n, every other one turned round
#pragma unroll
    for (int s = n >> 1; s > 0; s >>= 1) {
      const V ov = __shfl_xor_sync(0xffffffffu, v, s);
      const int oi = __shfl_xor_sync(0xffffffffu, i, s);
      const bool first = ((lane & s) == 0) == ((lane & n) == 0);
      if (better(ov, oi, v, i) == first) {
        v = ov;
        i = oi;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// selection, launch 1: a piece of a row per CTA
// ---------------------------------------------------------------------------
constexpr int kSelThreads = 256;         // that read logits; one more warp brings them in
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelBlock = kSelThreads + 32;
constexpr int kSelVecs = 8;              // 16-byte vectors of a thread at a time
constexpr int kSelStage = kSelThreads * kSelVecs * 16;   // bytes of all threads'
constexpr int kHeap = 512;               // candidates of a piece outside the lists
constexpr int kSelStages = 3;            // on their way, or being read
// A lane's sum is rescaled when its maximum has grown by this much: what was
// summed before then soon weighs nothing, and with it its rescalings' errors (a
// row in ascending order would rescale every round, 4e-5 over 2^24 values).
constexpr float kSelLag = 4.0f;

// A piece's sum of exp(l - max).
struct PieceSum {
  double sum;
  float max;
  float pad;
};

// signed integers in the order of the floats (NaN aside)
__device__ __forceinline__ int float_key(float x) {
  const int k = __float_as_int(x);
  return k ^ ((k >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float key_float(int k) {
  return __int_as_float(k ^ ((k >> 31) & 0x7fffffff));
}
__device__ __forceinline__ void readers_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(kSelThreads) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kSelBlock, 2)
    beam_piece_kernel(const __grid_constant__ BeamSelectArgs a, int pieces,
                      PieceSum* __restrict__ sums, float* __restrict__ vals,
                      int* __restrict__ ids) {
  using S = Storage<T>;
  constexpr int E = S::kVec;
  __shared__ float s_val[kSelWarps][32];
  __shared__ int s_id[kSelWarps][32];
  __shared__ double s_sum[kSelWarps];
  __shared__ float s_max[kSelWarps];
  extern __shared__ __align__(16) unsigned char ring[];   // [kSelStages][kSelStage]
  __shared__ uint64_t full[kSelStages], empty[kSelStages];
  __shared__ uint4 s_edge[kSelWarps];
  __shared__ float heap_val[kHeap];        // candidates, in no order
  __shared__ int heap_id[kHeap];
  __shared__ int s_heaped;                 // places given out, of any number
  __shared__ int s_bad;                    // a wait ran out
  __shared__ int s_bound;                  // key of a value that K values of the piece reach
  const int64_t row = blockIdx.y;
  const int piece = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_release();
  if (a.finished != nullptr && a.finished[row]) return;   // the merge does not read its pieces

  // The row's whole 16-byte vectors, cut evenly; its first piece also has the
  // elements before them, its last those behind.
  const T* base = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int vocab = static_cast<int>(a.vocab);
  const int head = min(vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) /
                                  static_cast<int>(sizeof(T)));
  const int vecs = (vocab - head) / E;
  const int v0 = static_cast<int>(static_cast<int64_t>(vecs) * piece / pieces);
  const int v1 = static_cast<int>(static_cast<int64_t>(vecs) * (piece + 1) / pieces);
  const uint4* whole = reinterpret_cast<const uint4*>(base + head);

  float m = kNegInf;                       // this lane's maximum, or up to kSelLag less
  double l = 0.0;                          // its sum about m
  float lv = kNegInf, worst = kNegInf;     // the warp's list: value, index of entry `lane`
  int li = kNoIndex;
  uint4 nothing;
  {
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = kNegInf;
    nothing = S::pack(f);
  }

  // kSelVecs vectors of every lane; the i-th has place i * kSelThreads + tid,
  // place p0 lies at from[0] in shared memory and begins at element id0 of the
  // row.  first: nothing is listed yet.
  auto take = [&](const uint4* raw, const uint4* from, int p0, int id0, bool first) {
    float vmax[kSelVecs], top = kNegInf;
#pragma unroll
    for (int i = 0; i < kSelVecs; ++i) {
      float f[E];
      S::unpack(raw[i], f);
      vmax[i] = fmaxf(f[0], f[1]);
#pragma unroll
      for (int e = 2; e < E; e += 2) vmax[i] = fmaxf(vmax[i], fmaxf(f[e], f[e + 1]));
      top = fmaxf(top, vmax[i]);
    }
    // a NaN makes the sum NaN, and so does +inf (inf - inf)
    if (top > m + kSelLag) {
      l = m == kNegInf ? l : l * static_cast<double>(ex2((m - top) * kLog2e));
      m = top;
    }
    const float about = m == kNegInf ? 0.0f : m;
    const uint64_t minus = pair_of(-about, -about), log2e = pair_of(kLog2e, kLog2e);
    uint64_t part[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kSelVecs; ++i) {
      float f[E];
      S::unpack(raw[i], f);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 z = halves_of(mul2(add2(pair_of(f[e], f[e + 1]), minus), log2e));
        part[(e >> 1) & 1] = add2(part[(e >> 1) & 1], pair_of(ex2(z.x), ex2(z.y)));
      }
    }
    const float2 sum2 = halves_of(add2(part[0], part[1]));
    l += static_cast<double>(sum2.x + sum2.y);
    if (first) {
      // The K-th largest of all lanes' maxima: every warp's K largest, then
      // every warp the K-th of those.
      const int lowest = static_cast<int>(0x80000000);
      int rest = float_key(top), kth = lowest;
      for (int k = 0; k < a.beams; ++k) {
        const int best = __reduce_max_sync(0xffffffffu, rest);
        const unsigned at = __ballot_sync(0xffffffffu, rest == best);
        if (lane == __ffs(at) - 1) rest = lowest;
        if (lane == k) kth = best;
      }
      s_id[warp][lane] = kth;
      readers_sync();
      int of[kSelWarps];
#pragma unroll
      for (int w = 0; w < kSelWarps; ++w) of[w] = s_id[w][lane];
      for (int k = 0; k < a.beams; ++k) {
        int mine = of[0];
#pragma unroll
        for (int w = 1; w < kSelWarps; ++w) mine = max(mine, of[w]);
        kth = __reduce_max_sync(0xffffffffu, mine);
        const unsigned at = __ballot_sync(0xffffffffu, mine == kth);
        if (lane == __ffs(at) - 1) {
          bool taken = false;
#pragma unroll
          for (int w = 0; w < kSelWarps; ++w)
            if (!taken && of[w] == kth) {
              of[w] = lowest;
              taken = true;
            }
        }
      }
      if (kth != lowest) {
        if (tid == 0) atomicMax(&s_bound, kth);
        worst = fmaxf(worst, key_float(max(kth - (kth == 0 ? 2 : 1), float_key(kNegInf))));
      }
    }
    // Values at or below what K listed values of any warp beat need no
    // listing; equal ones do, in case their index is lower, so worst stands
    // just below (the key below +0 is -0, which no comparison tells from it).
    const int shared = *reinterpret_cast<volatile int*>(&s_bound);
    worst = fmaxf(worst, key_float(max(shared - (shared == 0 ? 2 : 1), float_key(kNegInf))));
    unsigned mine = 0;                     // this lane's vectors that are worth a look
#pragma unroll
    for (int i = 0; i < kSelVecs; ++i) mine |= vmax[i] > worst ? 1u << i : 0u;
    // Such values are few: they go to the piece's heap, to be sorted at the
    // end, and a vector whose values have no room there to the warp's list.
    unsigned full_up = 0;
    for (unsigned look = mine; look; look &= look - 1) {
      const int i = __ffs(look) - 1, slot = i * kSelThreads + tid - p0;
      const T* x = reinterpret_cast<const T*>(from + slot);
      unsigned over = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) over |= S::to_float(x[e]) > worst ? 1u << e : 0u;
      int at = atomicAdd(&s_heaped, __popc(over));
      if (at + __popc(over) > kHeap) {
        full_up |= 1u << i;
        continue;
      }
      for (; over; over &= over - 1, ++at) {
        const int e = __ffs(over) - 1;
        heap_val[at] = S::to_float(x[e]);
        heap_id[at] = id0 + slot * E + e;
      }
    }
    mine = full_up;
    if (__ballot_sync(0xffffffffu, mine != 0) == 0) return;
    unsigned vectors = __reduce_or_sync(0xffffffffu, mine);
#pragma unroll 1
    while (vectors) {                      // in index order
      const int i = __ffs(vectors) - 1;
      vectors &= vectors - 1;
      unsigned todo = __ballot_sync(0xffffffffu, (mine >> i) & 1u);
#pragma unroll 1
      while (todo) {
        const int slot = i * kSelThreads + warp * 32 + __ffs(todo) - 1 - p0;
        todo &= todo - 1;
        const float v = lane < E ? S::to_float(reinterpret_cast<const T*>(from + slot)[lane])
                                 : kNegInf;
        unsigned hits = __ballot_sync(0xffffffffu, v > worst);
#pragma unroll 1
        while (hits) {
          const int e = __ffs(hits) - 1;
          const float x = __shfl_sync(0xffffffffu, v, e);
          const int place = __popc(__ballot_sync(0xffffffffu, lv >= x));
          const float uv = __shfl_up_sync(0xffffffffu, lv, 1);
          const int ui = __shfl_up_sync(0xffffffffu, li, 1);
          if (lane > place) {
            lv = uv;
            li = ui;
          } else if (lane == place) {
            lv = x;
            li = id0 + slot * E + e;
          }
          worst = fmaxf(worst, __shfl_sync(0xffffffffu, lv, a.beams - 1));
          hits &= hits - 1;
          hits &= __ballot_sync(0xffffffffu, v > worst);
        }
      }
    }
    const float last = __shfl_sync(0xffffffffu, lv, a.beams - 1);
    if (lane == 0 && last > kNegInf) atomicMax(&s_bound, float_key(last));
  };
  // elements [from, to) of the row, fewer than a vector's, as this warp's
  // lane 0's
  auto edge = [&](int from, int to) {
    uint4 raw[kSelVecs];
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      f[e] = lane == 0 && from + e < to ? S::to_float(base[from + e]) : kNegInf;
    raw[0] = S::pack(f);
#pragma unroll
    for (int i = 1; i < kSelVecs; ++i) raw[i] = nothing;
    if (lane == 0) s_edge[warp] = raw[0];
    __syncwarp();
    take(raw, s_edge + warp, warp * 32, from, false);
  };

  constexpr int kStep = kSelVecs * kSelThreads;
  const int rounds = max(1, (v1 - v0 + kStep - 1) / kStep);
  for (int k = tid; k < kHeap; k += kSelBlock) {
    heap_val[k] = kNegInf;
    heap_id[k] = kNoIndex;
  }
  if (tid == 0) {
    s_bound = float_key(kNegInf);
    s_heaped = 0;
    s_bad = 0;
    for (int k = 0; k < kSelStages; ++k) {
      mbarrier_init(&full[k], 1);
      mbarrier_init(&empty[k], kSelWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  if (warp == kSelWarps) {
    // ---- the piece's rounds, through a ring in shared memory ----
    for (int k = 0; k < rounds; ++k) {
      const int slot = k % kSelStages, n = min(kStep, v1 - v0 - k * kStep);
      if (k >= kSelStages && !mbarrier_wait(&empty[slot], ((k / kSelStages) & 1) ^ 1)) {
        if (lane == 0) s_bad = 1;
        for (int j = k - kSelStages; j < k; ++j)       // leave no copy in flight
          (void)mbarrier_wait(&full[j % kSelStages], (j / kSelStages) & 1);
        break;
      }
      const uint32_t dst = smem_addr(ring) + slot * kSelStage;
      const uint4* src = whole + v0 + static_cast<int64_t>(k) * kStep;
      if (n > 0 && elect_lane()) {
        mbarrier_expect(&full[slot], n * 16);
        bulk_load(dst, src, n * 16, &full[slot]);
      }
      __syncwarp();
      if (k + 1 < rounds && k >= kSelStages) {
        // Raise the bound: the K-th best of what is on the heap by now (what
        // is still being written there counts as -inf).
        const int on_heap = min(*reinterpret_cast<volatile int*>(&s_heaped), 64);
        float best = kNegInf;
        int none = kNoIndex;
        for (int j = 0; j < on_heap; j += 32) {
          float x = *reinterpret_cast<volatile float*>(&heap_val[j + lane]);
          int id = kNoIndex;
          sort_list(x, id, lane);
          merge_lists(best, none, x, id, lane);
        }
        const float last = __shfl_sync(0xffffffffu, best, a.beams - 1);
        if (lane == 0 && last > kNegInf) atomicMax(&s_bound, float_key(last));
        __syncwarp();
      }
    }
    return;
  }

  if (piece == 0 && warp == 0 && head > 0) edge(0, head);
#pragma unroll 1
  for (int k = 0; k < rounds; ++k) {
    const int at = v0 + k * kStep, slot = k % kSelStages;
    if (at < v1 && !mbarrier_wait(&full[slot], (k / kSelStages) & 1)) s_bad = 1;
    const uint4* stage = reinterpret_cast<const uint4*>(ring + slot * kSelStage);
    uint4 raw[kSelVecs];
#pragma unroll
    for (int i = 0; i < kSelVecs; ++i) {
      const int j = i * kSelThreads + tid;
      raw[i] = at + j < v1 ? stage[j] : nothing;
    }
    take(raw, stage, 0, head + at * E, k == 0);
    __syncwarp();
    if (lane == 0) mbarrier_arrive(&empty[slot]);
  }
  if (piece == pieces - 1 && warp == kSelWarps - 1 && head + vecs * E < vocab)
    edge(head + vecs * E, vocab);

  // the warp's maximum and sum
  const float wm = key_float(__reduce_max_sync(0xffffffffu, float_key(m)));
  double sum = l == 0.0 ? 0.0 : l * static_cast<double>(ex2((m - wm) * kLog2e));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) {
    s_sum[warp] = sum;
    s_max[warp] = wm;
  }
  readers_sync();
  // the heap into the lists, 32 candidates at a time; unless it ran over, no
  // other list has entries
  const int heaped = s_heaped;
  for (int at = warp * 32; at < min(heaped, kHeap); at += kSelThreads) {
    float x = heap_val[at + lane];
    int id = heap_id[at + lane];
    sort_list(x, id, lane);
    merge_lists(lv, li, x, id, lane);
  }
  int n = kSelWarps / 2;
  while (n > 0 && 32 * n >= heaped) n >>= 1;
  if (n > 0) {
    s_val[warp][lane] = lv;
    s_id[warp][lane] = li;
    readers_sync();
  }
#pragma unroll 1
  for (; n > 0; n >>= 1) {
    if (warp < n) {
      merge_lists(lv, li, s_val[warp + n][lane], s_id[warp + n][lane], lane);
      s_val[warp][lane] = lv;
      s_id[warp][lane] = li;
    }
    if (n > 1) readers_sync();
  }
  if (warp != 0) return;
  const int64_t at = row * pieces + piece;
  if (lane < a.beams) {
    vals[at * a.beams + lane] = lv;
    ids[at * a.beams + lane] = li;
  }
  float cm = lane < kSelWarps ? s_max[lane] : kNegInf;
  double cs = lane < kSelWarps ? s_sum[lane] : 0.0;
  const float top = warp_max(cm);
  cs = cs == 0.0 ? 0.0 : cs * static_cast<double>(ex2((cm - top) * kLog2e));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) cs += __shfl_xor_sync(0xffffffffu, cs, o);
  // (a failed piece offers nothing)
  if (lane == 0 && s_bad && a.status) atomicOr(a.status, VL_STATUS_TIMEOUT);
  if (lane == 0) sums[at] = PieceSum{s_bad ? static_cast<double>(NAN) : cs, top, 0.0f};
}

// ---------------------------------------------------------------------------
// selection, launch 2: an entry per CTA
// ---------------------------------------------------------------------------
constexpr int kMergeWarps = 8;

__global__ void __launch_bounds__(kMergeWarps * 32)
    beam_merge_kernel(const __grid_constant__ BeamSelectArgs a, int pieces,
                      const PieceSum* __restrict__ sums, const float* __restrict__ vals,
                      const int* __restrict__ ids) {
  __shared__ double s_val[VL_BEAM_MAX][32];
  __shared__ int s_id[VL_BEAM_MAX][32];
  const int64_t entry = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  for (int b = warp; b < a.beams; b += kMergeWarps) {
    const int64_t row = entry * a.beams + b;
    const double score = a.scores[row];
    double dv = -INFINITY;
    int di = kNoIndex;
    if (a.finished != nullptr && a.finished[row]) {
      if (lane == 0 && score > -INFINITY) {
        dv = score;
        di = static_cast<int>(b * a.vocab + a.pad_id);
      }
    } else {
      float lv = kNegInf;
      int li = kNoIndex;
      for (int p = 0; p < pieces; ++p) {
        const int64_t at = (row * pieces + p) * a.beams + lane;
        float w = kNegInf;
        int j = kNoIndex;
        if (lane < a.beams) {
          w = __ldcg(vals + at);
          j = __ldcg(ids + at);
        }
        if (p == 0) {
          lv = w;
          li = j;
        } else {
          merge_lists(lv, li, w, j, lane);
        }
      }
      // lse over the pieces: maximum, then the sums about it
      float m = kNegInf;
      for (int p = lane; p < pieces; p += 32) m = fmaxf(m, sums[row * pieces + p].max);
      m = warp_max(m);
      double sum = 0.0;
      for (int p = lane; p < pieces; p += 32) {
        const PieceSum ps = sums[row * pieces + p];
        if (ps.sum != 0.0) sum += ps.sum * static_cast<double>(ex2((ps.max - m) * kLog2e));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const double lse = static_cast<double>(m) + log(sum);
      const double v = score + static_cast<double>(lv) - lse;
      if (lane < a.beams && lv > kNegInf && isfinite(lse) && v > -INFINITY) {
        dv = v;
        di = static_cast<int>(b * a.vocab + li);
      }
    }
    s_val[b][lane] = dv;
    s_id[b][lane] = di;
  }
  __syncthreads();
  for (int n = 1; n < a.beams; n <<= 1) {
    for (int b = warp * 2 * n; b + n < a.beams; b += kMergeWarps * 2 * n) {
      double dv = s_val[b][lane];
      int di = s_id[b][lane];
      merge_lists(dv, di, s_val[b + n][lane], s_id[b + n][lane], lane);
      s_val[b][lane] = dv;
      s_id[b][lane] = di;
    }
    __syncthreads();
  }
  if (warp != 0) return;
  // every input of this entry has been read: outputs may be the inputs
  const double dv = s_val[0][lane];
  const int di = s_id[0][lane];
  int parent = lane;
  int64_t token = a.pad_id;
  bool done = true;
  if (lane < a.beams && di != kNoIndex) {
    const int vocab = static_cast<int>(a.vocab);
    parent = di / vocab;
    token = di - parent * vocab;
    done = a.finished != nullptr && a.finished[entry * a.beams + parent];
    for (int e = 0; e < a.n_eos; ++e) done = done || token == a.eos[e];
  }
  __syncwarp();
  if (lane < a.beams) {
    const int64_t at = entry * a.beams + lane;
    a.tokens[at] = token;
    a.parents[at] = parent;
    a.scores_out[at] = static_cast<float>(dv);
    if (a.finished_out != nullptr) a.finished_out[at] = done ? 1 : 0;
  }
}

// Pieces of a row: two CTAs per SM keep the memory busy, and what a piece
// costs by itself (first bound, lists, merges: several microseconds) speaks for
// few, long ones; but at least one round of vectors each.  64 x 5 f32 rows of
// 51865, 320 for 296 places: 20.9 us in one piece each, 26.4 in two, 29.9 as
// one line of equal shares (each CTA then ends one row and begins another).
int select_pieces(int64_t rows, int64_t vocab, int elems_per_vec) {
  const int64_t round = static_cast<int64_t>(kSelThreads) * kSelVecs * elems_per_vec;
  const int64_t most = (vocab + round - 1) / round;
  const int64_t want = (static_cast<int64_t>(sm_count()) * 2 + rows - 1) / rows;
  const int64_t n = want < most ? want : most;
  return static_cast<int>(n < 1 ? 1 : n);
}

template <typename T>
cudaError_t select_typed(const BeamSelectArgs& a, void* workspace, cudaStream_t stream) {
  const int64_t rows = a.batch * a.beams;
  const int pieces = select_pieces(rows, a.vocab, Storage<T>::kVec);
  PieceSum* sums = static_cast<PieceSum*>(workspace);
  float* vals = reinterpret_cast<float*>(sums + rows * pieces);
  int* ids = reinterpret_cast<int*>(vals + rows * pieces * a.beams);
  constexpr int smem = kSelStages * kSelStage;
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(beam_piece_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  e = launch_kernel(beam_piece_kernel<T>,
                    dim3(static_cast<unsigned>(pieces), static_cast<unsigned>(rows)),
                    dim3(kSelBlock), smem, stream, false, a, pieces, sums, vals, ids);
  if (e != cudaSuccess) return e;
  return launch_kernel(beam_merge_kernel, dim3(static_cast<unsigned>(a.batch)),
                       dim3(kMergeWarps * 32), 0, stream, true, a, pieces,
                       static_cast<const PieceSum*>(sums), static_cast<const float*>(vals),
                       static_cast<const int*>(ids));
}

// ---------------------------------------------------------------------------
// reordering
// ---------------------------------------------------------------------------
constexpr int kReorderThreads = 256;
constexpr int kReorderAhead = 4;         // vectors of a thread in flight

template <typename Vec>
__global__ void __launch_bounds__(kReorderThreads)
    beam_reorder_kernel(const __grid_constant__ BeamReorderArgs a) {
  extern __shared__ unsigned int used[];   // bitmap of the entry's range
  __shared__ int s_len[VL_BEAM_MAX];       // positions of row i's parent (-1: bad)
  __shared__ int s_row[VL_BEAM_MAX];       // its row in the old tables
  __shared__ int s_part[VL_BEAM_MAX];      // source of a copy (-1: none)
  __shared__ int s_write[VL_BEAM_MAX];     // page of the next position
  __shared__ int s_bad;
  const int64_t entry = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31;
  const int shift = ilog2(a.page_size), mask = a.page_size - 1;
  const int words = (a.pool_pages + 31) / 32;
  const int64_t first = a.pool_start[entry];
  const bool range_ok = first >= 0 && first + a.pool_pages <= a.num_pages;

  for (int w = tid; w < words; w += kReorderThreads) used[w] = 0;
  if (tid == 0) s_bad = range_ok ? 0 : 1;
  __syncthreads();
  if (tid < a.beams) {
    const int64_t p = a.parents[entry * a.beams + tid];
    int len = -1;
    int row = 0;
    if (p >= 0 && p < a.beams) {
      row = static_cast<int>(p);
      len = a.kv_len[entry * a.beams + p];
      if (len < 0 || static_cast<int64_t>(len) > (static_cast<int64_t>(a.max_pages) << shift))
        len = -1;
    }
    if (len < 0) s_bad = 1;
    s_len[tid] = len;
    s_row[tid] = row;
  }
  __syncthreads();

  // whole pages: shared with the parent, marked in the bitmap, copied into
  // the new table by the entry's first CTA
  for (int k = tid; k < a.beams * a.max_pages; k += kReorderThreads) {
    const int i = k / a.max_pages, j = k - i * a.max_pages;
    const int whole = s_len[i] < 0 ? 0 : s_len[i] >> shift;
    int page = -1;
    if (j < whole) {
      page = a.page_table[(entry * a.beams + s_row[i]) * a.table_stride + j];
      if (page < 0 || page >= a.num_pages) {
        page = -1;
        s_bad = 1;
      } else if (range_ok && page >= first && page < first + a.pool_pages) {
        const int at = static_cast<int>(page - first);
        atomicOr(&used[at >> 5], 1u << (at & 31));
      }
    }
    if (blockIdx.x == 0) a.table_out[(entry * a.beams + i) * a.table_out_stride + j] = page;
  }
  __syncthreads();

  if (tid < 32) {
    const int len = lane < a.beams ? s_len[lane] : -1;
    const int at = len >> shift, fill = len < 0 ? 0 : len & mask;
    const bool open = len >= 0 && at < a.max_pages;
    int part = -1;
    if (open && fill > 0) {
      part = a.page_table[(entry * a.beams + s_row[lane]) * a.table_stride + at];
      if (part < 0 || part >= a.num_pages) {
        part = -1;
        s_bad = 1;
      }
    }
    const bool has_part = part >= 0;
    bool keep = has_part && range_ok && part >= first && part < first + a.pool_pages;
    if (keep) {
      const int bit = static_cast<int>(part - first);
      keep = ((used[bit >> 5] >> (bit & 31)) & 1u) == 0;
    }
    for (int i = 0; i < a.beams; ++i) {
      const int other = __shfl_sync(0xffffffffu, part, i);
      if (i < lane && other == part) keep = false;
    }
    __syncwarp();
    if (keep) {
      const int bit = static_cast<int>(part - first);
      atomicOr(&used[bit >> 5], 1u << (bit & 31));
    }
    __syncwarp();
    const bool need = open && !keep && (fill == 0 || has_part);
    const unsigned needs = __ballot_sync(0xffffffffu, need);
    const int my_rank = __popc(needs & ((1u << lane) - 1));
    const int wanted = __popc(needs);
    int fresh = -1, seen = 0;               // the my_rank-th free page of the range
    for (int w0 = 0; range_ok && w0 < words && seen < wanted; w0 += 32) {
      unsigned int free_bits = 0;
      if (w0 + lane < words) {
        free_bits = ~used[w0 + lane];
        const int left = a.pool_pages - (w0 + lane) * 32;
        if (left < 32) free_bits &= (1u << left) - 1;
      }
      int upto = __popc(free_bits);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += n;
      }
      const int total = __shfl_sync(0xffffffffu, upto, 31);
      const int before = upto - __popc(free_bits);
      for (int r = seen; r < wanted && r < seen + total; ++r) {
        const int k = r - seen;             // the k-th free page of these 32 words
        const unsigned holder = __ballot_sync(0xffffffffu, before <= k && k < upto);
        int page = 0;
        if (before <= k && k < upto)
          page = (w0 + lane) * 32 + static_cast<int>(__fns(free_bits, 0, k - before + 1));
        page = __shfl_sync(0xffffffffu, page, __ffs(holder) - 1);
        if (need && my_rank == r) fresh = static_cast<int>(first) + page;
      }
      seen += total;
    }
    const int write = keep ? part : fresh;
    if (need && fresh < 0) s_bad = 1;
    if (lane < a.beams) {
      s_write[lane] = write;
      s_part[lane] = need && fresh >= 0 && has_part ? part : -1;
      if (blockIdx.x == 0) {
        if (open) a.table_out[(entry * a.beams + lane) * a.table_out_stride + at] = write;
        a.kv_len_out[entry * a.beams + lane] = len < 0 ? 0 : len;
      }
    }
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0 && s_bad && a.status) atomicOr(a.status, VL_STATUS_BAD_PAGE);

  // copies: (row, cache, layer) segments of fill rows, dealt to the CTAs
  int dealt = 0;
  for (int i = 0; i < a.beams; ++i) {
    const int part = s_part[i];
    if (part < 0) continue;
    const int64_t vecs = (s_len[i] & mask) * a.row_bytes / static_cast<int64_t>(sizeof(Vec));
    const int64_t segs = 2 * a.layers;
    const int64_t from = part * a.page_stride_bytes, to = s_write[i] * a.page_stride_bytes;
    int64_t s = static_cast<int64_t>(blockIdx.x) - dealt % gridDim.x;
    if (s < 0) s += gridDim.x;
    for (; s < segs; s += gridDim.x) {
      char* cache = static_cast<char*>(s < a.layers ? a.k_cache : a.v_cache) +
                    (s < a.layers ? s : s - a.layers) * a.layer_stride_bytes;
      const Vec* src = reinterpret_cast<const Vec*>(cache + from);
      Vec* dst = reinterpret_cast<Vec*>(cache + to);
      for (int64_t v = tid; v < vecs; v += kReorderAhead * kReorderThreads) {
        Vec x[kReorderAhead];
#pragma unroll
        for (int u = 0; u < kReorderAhead; ++u)
          if (v + u * kReorderThreads < vecs) x[u] = src[v + u * kReorderThreads];
#pragma unroll
        for (int u = 0; u < kReorderAhead; ++u)
          if (v + u * kReorderThreads < vecs) dst[v + u * kReorderThreads] = x[u];
      }
    }
    dealt = static_cast<int>((dealt + segs) % gridDim.x);
  }
}

}  // namespace

size_t beam_select_workspace_bytes(int64_t batch, int beams, int64_t vocab) {
  // (f32 rows have the most pieces)
  const size_t n = static_cast<size_t>(batch) * beams *
                   select_pieces(batch * beams, vocab, Storage<float>::kVec);
  return n * sizeof(PieceSum) + n * beams * (sizeof(float) + sizeof(int));
}

cudaError_t launch_beam_select(const BeamSelectArgs& a, int dtype, void* workspace,
                               cudaStream_t stream) {
  if (a.batch == 0) return cudaSuccess;
  switch (dtype) {
    case kDtypeF32: return select_typed<float>(a, workspace, stream);
    case kDtypeF16: return select_typed<__half>(a, workspace, stream);
    default: return select_typed<__nv_bfloat16>(a, workspace, stream);
  }
}

cudaError_t launch_beam_reorder(const BeamReorderArgs& a, cudaStream_t stream) {
  if (a.batch == 0) return cudaSuccess;
  // about eight CTAs per SM over the entries (32 x 5 rows, 28 layers: 23.6 us,
  // with four 26.2), and no more than there are segments when half the rows
  // copy
  int64_t per = (static_cast<int64_t>(sm_count()) * 8 + a.batch - 1) / a.batch;
  const int64_t most = 2 * a.layers * (a.beams > 1 ? a.beams / 2 : 1);
  if (per > most) per = most;
  if (per < 1) per = 1;
  const dim3 grid(static_cast<unsigned>(per), static_cast<unsigned>(a.batch));
  const size_t smem = static_cast<size_t>((a.pool_pages + 31) / 32) * 4;
  const uintptr_t all = reinterpret_cast<uintptr_t>(a.k_cache) |
                        reinterpret_cast<uintptr_t>(a.v_cache) |
                        static_cast<uintptr_t>(a.row_bytes) |
                        static_cast<uintptr_t>(a.page_stride_bytes) |
                        static_cast<uintptr_t>(a.layer_stride_bytes);
  if (all % 16 == 0)
    beam_reorder_kernel<uint4><<<grid, kReorderThreads, smem, stream>>>(a);
  else if (all % 4 == 0)
    beam_reorder_kernel<uint32_t><<<grid, kReorderThreads, smem, stream>>>(a);
  else
    beam_reorder_kernel<uint16_t><<<grid, kReorderThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace vl
