// Beam search for sm_100a: the selection of the best continuations over
// beams and vocabulary, and the reordering of paged caches after it.
//
// Selection.  A live beam b offers token v at s_b + l_bv - lse_b with
// lse_b = log sum_v exp(l_bv); the entry keeps the `beams` largest values,
// ties to the lower b * vocab + v.  Within a row the order is that of the
// logits, so the logits are read once: a row is cut into pieces that fit the
// registers of one CTA, which finds the piece's maximum, its sum of
// exponentials about that maximum and its `beams` largest logits; a second
// launch merges the pieces of the rows and the rows of an entry.  It is
// bound by the read of the logits, or for one entry by two launches'
// latency.
//   * Largest logits of a warp: the K-th largest of the 32 lane maxima is a
//     lower bound of the warp's K-th largest value, and few values reach it;
//     only the vectors that do are looked at element by element and
//     inserted into a list held one entry per lane.  Values are visited in
//     index order, so equal ones keep it.
//   * Lists are merged pairwise as bitonic sequences, five exchanges each.
//   * exp is evaluated on l - max of the lane's own values, summed in fp32
//     per lane (at most 64 terms) and in fp64 above that, and values are
//     compared in fp64: beams are told apart to about 1e-7.
//
// Reordering.  See vl_paged_beam_reorder in vl_api.h for the rule.  Every
// CTA of an entry works the small plan out for itself (a bitmap of the
// entry's range in shared memory), so one launch does tables and copies and
// nothing waits for another CTA.
#include <cmath>

#include "vl_common.cuh"
#include "vl_kernels.h"
#include "vl_paged.cuh"

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

// ---------------------------------------------------------------------------
// selection, launch 1: a piece of a row per CTA
// ---------------------------------------------------------------------------
constexpr int kSelThreads = 256;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelVecs = 8;              // 16-byte vectors a thread holds

// A piece's result: its largest logits and sum of exp(l - max).
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

template <typename T>
__global__ void __launch_bounds__(kSelThreads)
    beam_piece_kernel(const __grid_constant__ BeamSelectArgs a, int pieces, int64_t piece_vecs,
                      PieceSum* __restrict__ sums, float* __restrict__ vals,
                      int* __restrict__ ids) {
  using S = Storage<T>;
  constexpr int E = S::kVec;
  __shared__ float s_val[kSelWarps][32];
  __shared__ int s_id[kSelWarps][32];
  __shared__ double s_sum[kSelWarps];
  __shared__ float s_max[kSelWarps];
  const int64_t row = blockIdx.y;
  const int piece = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_release();
  if (a.finished != nullptr && a.finished[row]) return;   // the merge does not read its pieces

  // The row as 16-byte vectors from the boundary at or below its start;
  // vectors that reach outside the row are read element by element.
  const T* base = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int mis = static_cast<int>((reinterpret_cast<uintptr_t>(base) & 15) / sizeof(T));
  const T* first = base - mis;
  const int64_t end = a.vocab + mis;       // vector elements [mis, end) are the row's
  const int64_t v0 = static_cast<int64_t>(piece) * piece_vecs;
  const int64_t v1 = min(v0 + piece_vecs, (end + E - 1) / E);
  uint4 raw[kSelVecs];
  float vmax[kSelVecs];
#pragma unroll
  for (int i = 0; i < kSelVecs; ++i) {
    const int64_t j = v0 + i * kSelThreads + tid;
    const int64_t e0 = j * E;
    if (j < v1 && e0 >= mis && e0 + E <= end) {
      raw[i] = ld_stream(first + e0);
    } else {
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e)
        f[e] = j < v1 && e0 + e >= mis && e0 + e < end ? S::to_float(first[e0 + e]) : kNegInf;
      raw[i] = S::pack(f);
    }
  }
  float m = kNegInf;
#pragma unroll
  for (int i = 0; i < kSelVecs; ++i) {
    float f[E];
    S::unpack(raw[i], f);
    float x = f[0];
#pragma unroll
    for (int e = 1; e < E; ++e) x = fmaxf(x, f[e]);
    vmax[i] = x;
    m = fmaxf(m, x);
  }
  // a NaN makes the sum NaN, +inf makes it NaN too (inf - inf)
  float l = 0.0f;
#pragma unroll
  for (int i = 0; i < kSelVecs; ++i) {
    float f[E];
    S::unpack(raw[i], f);
#pragma unroll
    for (int e = 0; e < E; ++e)
      l += f[e] == kNegInf ? 0.0f : exp2f((f[e] - m) * 1.44269504f);
  }

  // the warp's maximum, sum and K-th largest lane maximum
  const int key = float_key(m);
  const float wm = key_float(__reduce_max_sync(0xffffffffu, key));
  double sum = l == 0.0f ? 0.0 : static_cast<double>(l) * exp2(static_cast<double>(m - wm) * 1.4426950408889634);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  int rest = key, bound = key;
  for (int k = 0; k < a.beams; ++k) {
    bound = __reduce_max_sync(0xffffffffu, rest);
    if (k + 1 == a.beams) break;
    const unsigned at = __ballot_sync(0xffffffffu, rest == bound);
    if (lane == __ffs(at) - 1) rest = static_cast<int>(0x80000000);
  }
  // (with K = 32 the last of them; lanes already taken out count lowest)
  const float floor_val = bound == static_cast<int>(0x80000000) ? kNegInf : key_float(bound);

  float lv = kNegInf;
  int li = kNoIndex;
  float worst = kNegInf;
#pragma unroll
  for (int i = 0; i < kSelVecs; ++i) {
    unsigned todo = __ballot_sync(0xffffffffu, vmax[i] >= floor_val && vmax[i] > worst);
    while (todo) {
      const int src = __ffs(todo) - 1;
      todo &= todo - 1;
      uint4 w;
      w.x = __shfl_sync(0xffffffffu, raw[i].x, src);
      w.y = __shfl_sync(0xffffffffu, raw[i].y, src);
      w.z = __shfl_sync(0xffffffffu, raw[i].z, src);
      w.w = __shfl_sync(0xffffffffu, raw[i].w, src);
      float f[E];
      S::unpack(w, f);
      const int64_t e0 = (v0 + i * kSelThreads + warp * 32 + src) * E - mis;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (f[e] > worst && f[e] >= floor_val) {       // warp-uniform
          const int place = __popc(__ballot_sync(0xffffffffu, lv >= f[e]));
          const float uv = __shfl_up_sync(0xffffffffu, lv, 1);
          const int ui = __shfl_up_sync(0xffffffffu, li, 1);
          if (lane > place) {
            lv = uv;
            li = ui;
          } else if (lane == place) {
            lv = f[e];
            li = static_cast<int>(e0 + e);
          }
          worst = __shfl_sync(0xffffffffu, lv, a.beams - 1);
        }
      }
    }
  }
  s_val[warp][lane] = lv;
  s_id[warp][lane] = li;
  if (lane == 0) {
    s_sum[warp] = sum;
    s_max[warp] = wm;
  }
  __syncthreads();
#pragma unroll
  for (int n = kSelWarps / 2; n > 0; n >>= 1) {
    if (warp < n) {
      merge_lists(lv, li, s_val[warp + n][lane], s_id[warp + n][lane], lane);
      s_val[warp][lane] = lv;
      s_id[warp][lane] = li;
    }
    if (n > 1) __syncthreads();
  }
  if (warp != 0) return;
  const int64_t at = row * pieces + piece;
  if (lane < a.beams) {
    vals[at * a.beams + lane] = lv;
    ids[at * a.beams + lane] = li;
  }
  if (lane == 0) {
    float cm = s_max[0];
    for (int w = 1; w < kSelWarps; ++w) cm = fmaxf(cm, s_max[w]);
    double cs = 0.0;
    for (int w = 0; w < kSelWarps; ++w)
      cs += s_sum[w] == 0.0 ? 0.0 : s_sum[w] * exp2(static_cast<double>(s_max[w] - cm) * 1.4426950408889634);
    sums[at] = PieceSum{cs, cm, 0.0f};
  }
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
        if (ps.sum != 0.0) sum += ps.sum * exp2(static_cast<double>(ps.max - m) * 1.4426950408889634);
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
    parent = static_cast<int>(di / a.vocab);
    token = di % a.vocab;
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

// Pieces of a row: as many as its vectors need at kSelVecs per thread, cut
// evenly.
void select_pieces(int64_t vocab, int elems_per_vec, int* pieces, int64_t* piece_vecs) {
  const int64_t vecs = (vocab + elems_per_vec - 1) / elems_per_vec + 1;   // a misaligned row has one more
  const int64_t hold = static_cast<int64_t>(kSelThreads) * kSelVecs;
  const int64_t n = (vecs + hold - 1) / hold;
  *pieces = static_cast<int>(n);
  *piece_vecs = (vecs + n - 1) / n;
}

template <typename T>
cudaError_t select_typed(const BeamSelectArgs& a, void* workspace, cudaStream_t stream) {
  int pieces;
  int64_t piece_vecs;
  select_pieces(a.vocab, Storage<T>::kVec, &pieces, &piece_vecs);
  const int64_t rows = a.batch * a.beams;
  PieceSum* sums = static_cast<PieceSum*>(workspace);
  float* vals = reinterpret_cast<float*>(sums + rows * pieces);
  int* ids = reinterpret_cast<int*>(vals + rows * pieces * a.beams);
  beam_piece_kernel<T><<<dim3(static_cast<unsigned>(pieces), static_cast<unsigned>(rows)),
                         kSelThreads, 0, stream>>>(a, pieces, piece_vecs, sums, vals, ids);
  cudaError_t e = cudaGetLastError();
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
  for (int i = 0; i < a.beams; ++i) {
    const int whole = s_len[i] < 0 ? 0 : s_len[i] >> shift;
    const int32_t* src = a.page_table + (entry * a.beams + s_row[i]) * a.table_stride;
    int32_t* dst = a.table_out + (entry * a.beams + i) * a.table_out_stride;
    for (int j = tid; j < a.max_pages; j += kReorderThreads) {
      int page = -1;
      if (j < whole) {
        page = src[j];
        if (page < 0 || page >= a.num_pages) {
          page = -1;
          s_bad = 1;
        } else if (range_ok && page >= first && page < first + a.pool_pages) {
          const int at = static_cast<int>(page - first);
          atomicOr(&used[at >> 5], 1u << (at & 31));
        }
      }
      if (blockIdx.x == 0) dst[j] = page;
    }
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
      for (int64_t v = tid; v < vecs; v += 4 * kReorderThreads) {
        Vec x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (v + u * kReorderThreads < vecs) x[u] = src[v + u * kReorderThreads];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (v + u * kReorderThreads < vecs) dst[v + u * kReorderThreads] = x[u];
      }
    }
    dealt = static_cast<int>((dealt + segs) % gridDim.x);
  }
}

}  // namespace

size_t beam_select_workspace_bytes(int64_t batch, int beams, int64_t vocab) {
  int pieces;
  int64_t piece_vecs;
  select_pieces(vocab, Storage<float>::kVec, &pieces, &piece_vecs);   // the most pieces of any type
  const size_t n = static_cast<size_t>(batch) * beams * pieces;
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
  // about four CTAs per SM over the entries, and no more than there are
  // segments when every row but one copies
  int64_t per = (static_cast<int64_t>(sm_count()) * 4 + a.batch - 1) / a.batch;
  const int64_t most = 2 * a.layers * (a.beams > 1 ? a.beams - 1 : 1);
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
