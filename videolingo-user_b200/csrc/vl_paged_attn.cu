// Attention over a paged KV cache for sm_100a: the kernel of single and few
// new tokens, the kernel of the remaining types, and the choice between them
// and the tcgen05 kernel of longer chunks (vl_paged_attn_tc.cu).
//
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j,  j <= kv_len - n + i
//
// Few tokens.  With R = n * G <= 16 query rows per kv head (G query heads
// share it) the work is one read of the sequence's cached rows: bound by
// HBM.  The rows of q are the N of mma.sync m16n8k16 and the positions its
// M, so K and V go from shared memory to the tensor cores as they lie:
// S^T = K q^T, then O^T += V^T P^T with P^T from the accumulators by
// movmatrix.
//   * Balance: lengths differ and live on the device.  All (sequence, kv
//     head) pairs' tiles of 64 positions form one line of units, in order,
//     and every CTA takes an equal run of it, whatever pairs that crosses.
//     A pair that lies within one run is finished there; one that is cut
//     leaves partial sums (at most two per CTA), and a second launch, ready
//     before the first ends, joins them in order.  Neither grid nor
//     workspace depends on the lengths.  Short caches of few pairs take a
//     cluster of CTAs per pair instead, joined through distributed shared
//     memory, and no second launch.
//   * A producer warp turns page ids into TMA boxes (64 dims x up to 64 rows
//     of one page, 128-byte swizzle) and runs ahead of the four consumer
//     warps, across pairs, through a ring of 64-position stages.
//   * A consumer warp owns 16 positions of a stage and keeps its own running
//     maximum and sums; warps are joined once per pair.
// 64 sequences of up to 4096 positions (269 MB), 16 / 4 heads of 128: 53.5 us,
// 5.0 TB/s, 0.77 of the measured copy rate (90 us and 0.91 when all are that
// long); what is left is the ring's start and the join.  4 sequences of 500:
// 6.7 us, the latency of a launch, of lengths, pages and rows one after the
// other, and of the join.  Pages that beams share are read once per beam; most
// of that comes from L2 (16 x 4 beams of 421 positions 12.9 us, 16.9 with pages
// of their own; 32 x 5: 28.0 and 34.5).
#include <cudaTypedefs.h>

#include <atomic>
#include <cmath>

#include "vl_common.cuh"
#include "vl_kernels.h"
#include "vl_paged.cuh"
#include "vl_tma.cuh"

namespace vl {
namespace {

// ---------------------------------------------------------------------------
// tensor maps
// ---------------------------------------------------------------------------
using EncodeTiled = PFN_cuTensorMapEncodeTiled_v12000;

EncodeTiled encoder() {
  static std::atomic<EncodeTiled> fn{nullptr};
  EncodeTiled f = fn.load(std::memory_order_acquire);
  if (f != nullptr) return f;
  void* p = nullptr;
  cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
          cudaSuccess ||
      q != cudaDriverEntryPointSuccess || p == nullptr) {
    (void)cudaGetLastError();
    return nullptr;
  }
  f = reinterpret_cast<EncodeTiled>(p);
  fn.store(f, std::memory_order_release);
  return f;
}

// ---------------------------------------------------------------------------
// few new tokens
// ---------------------------------------------------------------------------
constexpr int kFewRows = 16;              // query rows per kv head, at most
constexpr int kFewTile = 64;              // positions of a unit
constexpr int kFewWarps = 4;              // consumer warps
constexpr int kFewThreads = (kFewWarps + 1) * 32;
constexpr int kFewStages = 3;
constexpr int kFewCtasPerSm = 2;
constexpr int kFewCluster = 4;            // CTAs of a pair, where a cluster takes one
// Weights are held times 2^15 in f16, the largest that it takes: small ones keep
// their bits down to 2^-29 of the largest and some down to 2^-39, where sums of
// thousands of them count beside one large weight.  bf16 has fp32's exponents.
template <typename T>
constexpr float kFewLift = std::is_same<T, __half>::value ? 15.0f : 0.0f;

__host__ __device__ constexpr int few_partial_floats(int hd) { return kFewRows * hd + 2 * kFewRows; }

// Device-side view of the workspace.
struct FewWork {
  int64_t* base;      // [batch + 2]: units before each sequence, their total, units per CTA
  float* part;        // [2 * grid]: rows [16][hd], then (max, sum) pairs
};

// Where a run of units lies: sequence, its units before, its tiles per head.
struct Cursor {
  int b;
  int64_t base;
  SeqView s;
  int tiles;
};

template <typename T, int HD, int NT>
struct FewSmem {
  float wm[kFewWarps][8 * NT];
  float wl[kFewWarps][8 * NT];
  float part[2][8][HD + 4];
  uint64_t full[kFewStages];
  uint64_t empty[kFewStages];
  int bad;                                // a wait ran out
  int stop;                               // bad, as all consumers read it at a pair's end
};

__device__ __forceinline__ void few_sync() {   // the consumer warps
  asm volatile("bar.sync 1, %0;" ::"n"(kFewWarps * 32) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                      uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ int few_tiles(const SeqView& s) {
  return s.rows > 0 ? (s.len + kFewTile - 1) / kFewTile : 0;
}

// Total units, and the cursor of unit `u` (a whole warp; lane l adds up the
// l-th 32nd of the sequences).  With `base` the units before each sequence
// are written down.
__device__ __forceinline__ int64_t few_total(const PagedAttnArgs& a, int shift, int lane,
                                             int64_t* before, int64_t* base) {
  const int each = (a.batch + 31) / 32;
  const int b0 = min(a.batch, lane * each), b1 = min(a.batch, b0 + each);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b)
    mine += static_cast<int64_t>(few_tiles(sequence_view(a, b, shift))) * a.n_kv_heads;
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t n = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += n;
  }
  *before = upto - mine;
  if (base != nullptr) {
    int64_t at = upto - mine;
    for (int b = b0; b < b1; ++b) {
      base[b] = at;
      at += static_cast<int64_t>(few_tiles(sequence_view(a, b, shift))) * a.n_kv_heads;
    }
  }
  return __shfl_sync(0xffffffffu, upto, 31);
}

__device__ __forceinline__ Cursor few_locate(const PagedAttnArgs& a, int shift, int lane,
                                             int64_t before, int64_t u) {
  // the last lane whose sequences begin at or before u holds it
  const int owner = 31 - __clz(__ballot_sync(0xffffffffu, before <= u));
  Cursor c;
  c.b = owner * ((a.batch + 31) / 32);
  c.base = __shfl_sync(0xffffffffu, before, owner);
  for (;; ++c.b) {
    if (c.b >= a.batch) break;
    c.s = sequence_view(a, c.b, shift);
    c.tiles = few_tiles(c.s);
    const int64_t n = static_cast<int64_t>(c.tiles) * a.n_kv_heads;
    if (u < c.base + n) break;
    c.base += n;
  }
  return c;
}
// The next sequence with anything to do.
__device__ __forceinline__ void few_next(const PagedAttnArgs& a, int shift, Cursor& c) {
  c.base += static_cast<int64_t>(c.tiles) * a.n_kv_heads;
  do {
    ++c.b;
    if (c.b >= a.batch) return;
    c.s = sequence_view(a, c.b, shift);
    c.tiles = few_tiles(c.s);
  } while (c.tiles == 0);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// The shared-memory address of block `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
  uint32_t y;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(y) : "r"(addr), "r"(rank));
  return y;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
  float4 y;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w)
               : "r"(addr)
               : "memory");
  return y;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t addr) {
  float2 y;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(y.x), "=f"(y.y) : "r"(addr)
               : "memory");
  return y;
}

// C = 1: a run of the line of units.  C > 1: a cluster of C CTAs per pair, an
// equal share of its tiles each, joined through distributed shared memory.
template <typename T, int HD, int NT, int C>
__device__ __forceinline__ void few_body(const PagedAttnArgs& a, const CUtensorMap& kmap,
                                         const CUtensorMap& vmap, const FewWork& work,
                                         int box_shift) {
  using S = Storage<T>;
  constexpr int KS = HD / 16;             // k-steps of q.k, m-tiles of p.v
  constexpr int kHalves = HD / 64;        // 128-byte columns of a row
  constexpr int kColumn = kFewTile * 128; // bytes of one
  constexpr int kMatrix = kHalves * kColumn;
  constexpr int kStage = 2 * kMatrix;     // K, then V
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw0 = smem_addr(smem_raw);
  const uint32_t ring = (raw0 + 1023) & ~1023u;   // the swizzle counts from 1 KB boundaries
  FewSmem<T, HD, NT>& sm = *reinterpret_cast<FewSmem<T, HD, NT>*>(
      smem_raw + (ring - raw0) + kFewStages * kStage);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int shift = ilog2(a.page_size);
  const int G = a.n_q_heads / a.n_kv_heads;
  if (tid == kFewWarps * 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kmap)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&vmap)) : "memory");
  }
  if (tid == 0) {
    for (int s = 0; s < kFewStages; ++s) {
      mbarrier_init(&sm.full[s], 1);
      mbarrier_init(&sm.empty[s], kFewWarps);
    }
    sm.bad = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // lengths and tables are not written by the kernel before this one; the
  // tables are on their way to L2 while the lengths are added up
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kFewThreads + tid;
       i * 32 < a.batch * a.table_stride - (a.table_stride - a.max_pages);
       i += static_cast<int64_t>(gridDim.x) * kFewThreads)
    asm volatile("prefetch.global.L2 [%0];" ::"l"(a.page_table + i * 32));
  int64_t before = 0, total = 0, share = 0, u0, u1;
  const bool note = C == 1 && blockIdx.x == 0 && warp == 0;
  const int rank = C == 1 ? 0 : static_cast<int>(blockIdx.x % C);
  Cursor c;
  if (C == 1) {
    total = few_total(a, shift, lane, &before, nullptr);
    share = max(int64_t(1), divide(total + gridDim.x - 1, gridDim.x));
    u0 = blockIdx.x * share;
    u1 = min(total, u0 + share);
    c.b = a.batch;
    if (u0 < u1) c = few_locate(a, shift, lane, before, u0);
  } else {
    const int pair = blockIdx.x / C;
    c.b = pair / a.n_kv_heads;
    c.base = 0;
    c.s = sequence_view(a, c.b, shift);
    c.tiles = few_tiles(c.s);
    const int64_t first = static_cast<int64_t>(pair - c.b * a.n_kv_heads) * c.tiles;
    u0 = first + c.tiles * rank / C;
    u1 = first + c.tiles * (rank + 1) / C;
  }
  // the first tile's pages, for the producer
  const int box_rows = 1 << box_shift;
  auto pages_of = [&](int64_t u) {        // lane l: the l-th box's page
    const int local = static_cast<int>(u - c.base);
    const int pos0 = (local % c.tiles) * kFewTile;
    int page = 0;
    if (lane * box_rows < min(kFewTile, c.s.len - pos0)) {
      page = a.page_table[c.b * a.table_stride + ((pos0 + (lane << box_shift)) >> shift)];
      if (page < 0 || page >= a.num_pages) {            // read as rows of zeros
        page = static_cast<int>(a.num_pages);
        if (a.status) atomicOr(a.status, VL_STATUS_BAD_PAGE);
      }
    }
    return page;
  };
  int page = 0;
  if (warp == kFewWarps && u0 < u1) page = pages_of(u0);
  __syncthreads();
  pdl_wait();
  pdl_release();
  if (note) {
    few_total(a, shift, lane, &before, work.base);
    if (lane == 0) {
      work.base[a.batch] = total;
      work.base[a.batch + 1] = share;
    }
  }
  if (C > 1) {
    const int h = static_cast<int>(blockIdx.x / C) - c.b * a.n_kv_heads;
    if (c.s.bad && h == 0 && rank == 0 && tid == 0 && a.status)
      atomicOr(a.status, VL_STATUS_BAD_PAGE);
    if (c.tiles == 0) {                   // (the whole cluster)
      T* out = static_cast<T*>(a.out) + static_cast<int64_t>(c.s.start) * a.out_row_stride +
               static_cast<int64_t>(h) * G * HD;
      const int64_t vecs = static_cast<int64_t>(c.s.rows) * G * (HD / 8);
      for (int64_t i = rank * kFewThreads + tid; i < vecs; i += C * kFewThreads)
        st_vec(out + i / (G * (HD / 8)) * a.out_row_stride + i % (G * (HD / 8)) * 8,
               make_uint4(0, 0, 0, 0));
      return;
    }
  } else if (u0 >= u1) {
    return;
  }

  if (warp == kFewWarps) {
    // ---- producer ----
    int stage = 0;
    uint32_t phase = 0;
    int64_t issued = 0;
    for (int64_t u = u0; u < u1; ++u) {
      while (u >= c.base + static_cast<int64_t>(c.tiles) * a.n_kv_heads) few_next(a, shift, c);
      const int local = static_cast<int>(u - c.base);
      const int h = local / c.tiles, tile = local - h * c.tiles;
      const int pos0 = tile * kFewTile;
      const int need = (min(kFewTile, c.s.len - pos0) + box_rows - 1) >> box_shift;
      if (u != u0) page = pages_of(u);    // before the wait for the stage
      if (issued >= kFewStages && !mbarrier_wait(&sm.empty[stage], phase ^ 1)) {
        if (lane == 0) atomicExch(&sm.bad, 1);
        break;
      }
      if (elect_lane())
        mbarrier_expect(&sm.full[stage], static_cast<uint32_t>(need) * box_rows * 128 * kHalves * 2);
      __syncwarp();
      for (int j = 0; j < need; ++j) {
        const int pj = __shfl_sync(0xffffffffu, page, j);
        const uint32_t dst = ring + stage * kStage + j * box_rows * 128;
        const int row = (pos0 + (j << box_shift)) & (a.page_size - 1);
        if (elect_lane()) {
#pragma unroll
          for (int half = 0; half < kHalves; ++half) {
            tma_load_4d(dst + half * kColumn, &kmap, half * 64, h, row, pj, &sm.full[stage]);
            tma_load_4d(dst + half * kColumn + kMatrix, &vmap, half * 64, h, row, pj,
                        &sm.full[stage]);
          }
        }
        __syncwarp();
      }
      ++issued;
      if (++stage == kFewStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (*reinterpret_cast<volatile int*>(&sm.bad)) {
      // leave no copy in flight: the last one into each stage
      for (int64_t i = issued < kFewStages ? 0 : issued - kFewStages; i < issued; ++i)
        (void)mbarrier_wait(&sm.full[i % kFewStages], static_cast<uint32_t>((i / kFewStages) & 1));
    }
    return;
  }

  // ---- consumers ----
  const int gid = lane >> 2, tig = lane & 3, mi = lane >> 3;
  const int wrow = warp * 16;
  const float qscale = a.scale * kLog2e;
  int stage = 0;
  uint32_t phase = 0;
  int64_t u = u0;
  bool first_piece = true;
  while (u < u1) {
    while (u >= c.base + static_cast<int64_t>(c.tiles) * a.n_kv_heads) few_next(a, shift, c);
    const int local = static_cast<int>(u - c.base);
    const int h = local / c.tiles, t0 = local - h * c.tiles;
    const int t1 = static_cast<int>(min(static_cast<int64_t>(c.tiles), t0 + (u1 - u)));
    const int R = c.s.rows * G;

    uint32_t qb[NT][KS][2];               // q^T as the B operand: column n = row nt * 8 + gid
    int seen[NT][2];                      // positions that column nt * 8 + 2 tig + e sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int n = nt * 8 + gid;
      const bool ok = n < R;
      const T* qrow = static_cast<const T*>(a.q) +
                      static_cast<int64_t>(c.s.start + (ok ? n / G : 0)) * a.q_row_stride +
                      static_cast<int64_t>(h * G + (ok ? n % G : 0)) * HD + tig * 2;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qb[nt][ks][0] = ok ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16) : 0u;
        qb[nt][ks][1] = ok ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 8) : 0u;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = nt * 8 + 2 * tig + e;
        seen[nt][e] = col < R ? c.s.len - c.s.rows + col / G + 1 : 0;
      }
    }
    float m_run[NT][2], l_run[NT][2], o[NT][KS][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m_run[nt][e] = -INFINITY;
        l_run[nt][e] = 0.0f;
      }
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][ks][e] = 0.0f;
    }

    for (int tile = t0; tile < t1; ++tile) {
      if (!mbarrier_wait(&sm.full[stage], phase)) {
        if (lane == 0) atomicExch(&sm.bad, 1);
        break;
      }
      const uint32_t kt = ring + stage * kStage, vt = kt + kMatrix;
      const int pos0 = tile * kFewTile + wrow;
      if (pos0 < c.s.len) {
        if (pos0 + 16 > c.s.len) {
          // rows of V past the end hold anything: their weights are 0, and
          // so must they be
          for (int i = lane; i < 16 * KS * 2; i += 32) {
            const int r = i / (KS * 2), ch = i % (KS * 2);
            if (pos0 + r >= c.s.len)
              asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(
                               vt + (ch >> 3) * kColumn + (wrow + r) * 128 +
                               (((ch & 7) ^ ((wrow + r) & 7)) << 4)),
                           "r"(0)
                           : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        float sacc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sacc[nt][e] = 0.0f;
        {
          const int r = wrow + (mi & 1) * 8 + (lane & 7);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const int ch = ks * 2 + (mi >> 1);
            uint32_t af[4];
            ldmatrix4(af, kt + (ch >> 3) * kColumn + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16(sacc[nt], af, qb[nt][ks][0], qb[nt][ks][1], T());
          }
        }
        uint32_t pb[NT][2];
        float alpha[NT][2];
        bool rescale = false;
        const int p0 = pos0 + gid, p1 = p0 + 8;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float sv[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            sv[e] = p0 < seen[nt][e] ? sacc[nt][e] * qscale : -INFINITY;
            sv[e + 2] = p1 < seen[nt][e] ? sacc[nt][e + 2] * qscale : -INFINITY;
            float mt = fmaxf(sv[e], sv[e + 2]);
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 4));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 8));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 16));
            const float m_new = fmaxf(m_run[nt][e], mt);
            // nothing seen yet: -inf - -inf would be NaN
            alpha[nt][e] = m_new == -INFINITY ? 1.0f : exp2f(m_run[nt][e] - m_new);
            rescale |= alpha[nt][e] != 1.0f;
            m_run[nt][e] = m_new;
            // (lifted after the difference: scores past 2^24 have no room for it)
            sv[e] = sv[e] == -INFINITY ? 0.0f : exp2f(sv[e] - m_new + kFewLift<T>);
            sv[e + 2] = sv[e + 2] == -INFINITY ? 0.0f : exp2f(sv[e + 2] - m_new + kFewLift<T>);
            l_run[nt][e] = fmaf(l_run[nt][e], alpha[nt][e], sv[e] + sv[e + 2]);
          }
          // P rounds to the storage type, as its tensor-core operand: half a
          // step per weight, against sums that stay in fp32
          pb[nt][0] = transpose8(pack16(sv[0], sv[1], T()));
          pb[nt][1] = transpose8(pack16(sv[2], sv[3], T()));
        }
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              o[nt][ks][0] *= alpha[nt][0];
              o[nt][ks][1] *= alpha[nt][1];
              o[nt][ks][2] *= alpha[nt][0];
              o[nt][ks][3] *= alpha[nt][1];
            }
        }
        {
          const int r = wrow + (mi >> 1) * 8 + (lane & 7);
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            const int ch = ks * 2 + (mi & 1);
            uint32_t af[4];
            ldmatrix4_t(af, vt + (ch >> 3) * kColumn + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16(o[nt][ks], af, pb[nt][0], pb[nt][1], T());
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&sm.empty[stage]);
      if (++stage == kFewStages) {
        stage = 0;
        phase ^= 1;
      }
    }

    // ---- join the warps: common maximum, then sums in warp order ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l = l_run[nt][e];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (gid == 0) {
          sm.wm[warp][nt * 8 + 2 * tig + e] = m_run[nt][e];
          sm.wl[warp][nt * 8 + 2 * tig + e] = l;
        }
      }
    if (tid == 0) sm.stop = *reinterpret_cast<volatile int*>(&sm.bad);
    few_sync();
    const bool failed = sm.stop != 0;
    const bool whole = C == 1 && t0 == 0 && t1 == c.tiles;
    // (a cluster's lie where the ring was: its last stage has been read)
    const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (first_piece ? 0 : 1);
    float* part = C > 1 ? reinterpret_cast<float*>(smem_raw + (ring - raw0))
                        : work.part + slot * few_partial_floats(HD);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {     // eight rows at a time
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = nt * 8 + 2 * tig + e;
        float M = sm.wm[0][col];
#pragma unroll
        for (int w = 1; w < kFewWarps; ++w) M = fmaxf(M, sm.wm[w][col]);
        const float f = m_run[nt][e] == -INFINITY ? 0.0f : exp2f(m_run[nt][e] - M);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          o[nt][ks][e] *= f;
          o[nt][ks][e + 2] *= f;
        }
      }
      if (warp >= 2) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sm.part[warp - 2][2 * tig + (e & 1)][ks * 16 + gid + (e >> 1) * 8] = o[nt][ks][e];
      }
      few_sync();
      if (warp < 2) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            sm.part[warp][2 * tig + (e & 1)][ks * 16 + gid + (e >> 1) * 8] += o[nt][ks][e];
      }
      few_sync();
      const int rows = min(8, R - nt * 8);
      for (int i = tid; i < rows * (HD / 8); i += kFewWarps * 32) {
        const int r = i / (HD / 8), d = (i % (HD / 8)) * 8;
        const int n = nt * 8 + r;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = sm.part[0][r][d + e] + sm.part[1][r][d + e];
        float M = sm.wm[0][n];
#pragma unroll
        for (int w = 1; w < kFewWarps; ++w) M = fmaxf(M, sm.wm[w][n]);
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w)
          if (sm.wm[w][n] != -INFINITY) L = fmaf(sm.wl[w][n], exp2f(sm.wm[w][n] - M), L);
          else L += sm.wl[w][n];          // 0, or NaN where every score seen was NaN
        if (failed) L = __int_as_float(0x7fc00000);
        if (whole) {
          const float inv = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= inv;
          st_vec(static_cast<T*>(a.out) +
                     static_cast<int64_t>(c.s.start + n / G) * a.out_row_stride +
                     static_cast<int64_t>(h * G + n % G) * HD + d,
                 S::pack(f));
        } else {
          float4* dst = reinterpret_cast<float4*>(part + n * HD + d);
          dst[0] = make_float4(f[0], f[1], f[2], f[3]);
          dst[1] = make_float4(f[4], f[5], f[6], f[7]);
          if (d == 0)
            *reinterpret_cast<float2*>(part + kFewRows * HD + 2 * n) = make_float2(M, L);
        }
      }
      few_sync();                         // the shared sums are free again
    }
    if (failed) {
      if (tid == 0 && a.status) atomicOr(a.status, VL_STATUS_TIMEOUT);
      if (C == 1) return;
    }
    first_piece = false;
    u += t1 - t0;
  }
  if (C > 1) {
    // ---- join the cluster's pieces, in order: four dims of a row a thread ----
    const int h = static_cast<int>(blockIdx.x / C) - c.b * a.n_kv_heads, R = c.s.rows * G;
    if (u0 >= u1 && tid < kFewRows)
      reinterpret_cast<float2*>(smem_raw + (ring - raw0) + kFewRows * HD * 4)[tid] =
          make_float2(-INFINITY, 0.0f);
    cluster_sync();
    for (int i = tid * C + rank; i < R * (HD / 4); i += kFewWarps * 32 * C) {
      const int row = i / (HD / 4), d = i % (HD / 4) * 4;
      float2 ml[C];
      float4 x[C];
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const uint32_t at = cluster_addr(ring, k);
        ml[k] = cluster_load2(at + (kFewRows * HD + 2 * row) * 4);
        x[k] = cluster_load4(at + (row * HD + d) * 4);
      }
      float M = ml[0].x, L = 0.0f;
#pragma unroll
      for (int k = 1; k < C; ++k) M = fmaxf(M, ml[k].x);
      float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < C; ++k) {
        if (ml[k].x == -INFINITY && ml[k].y == 0.0f) continue;   // nothing seen, or no tiles
        const float w = ml[k].x == -INFINITY ? 1.0f : exp2f(ml[k].x - M);
        L = fmaf(ml[k].y, w, L);
        f.x = fmaf(x[k].x, w, f.x);
        f.y = fmaf(x[k].y, w, f.y);
        f.z = fmaf(x[k].z, w, f.z);
        f.w = fmaf(x[k].w, w, f.w);
      }
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      const uint2 y =
          make_uint2(pack16(f.x * inv, f.y * inv, T()), pack16(f.z * inv, f.w * inv, T()));
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) +
                                static_cast<int64_t>(c.s.start + row / G) * a.out_row_stride +
                                static_cast<int64_t>(h * G + row % G) * HD + d) = y;
    }
    cluster_sync();                       // nobody leaves while its sums are being read
  }
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(kFewThreads, kFewCtasPerSm)
    paged_few_kernel(const __grid_constant__ PagedAttnArgs a,
                     const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, FewWork work, int box_shift) {
  few_body<T, HD, NT, 1>(a, kmap, vmap, work, box_shift);
}
template <typename T, int HD, int NT, int C>
__global__ void __cluster_dims__(C, 1, 1) __launch_bounds__(kFewThreads, kFewCtasPerSm)
    paged_few_cluster_kernel(const __grid_constant__ PagedAttnArgs a,
                             const __grid_constant__ CUtensorMap kmap,
                             const __grid_constant__ CUtensorMap vmap, FewWork work,
                             int box_shift) {
  few_body<T, HD, NT, C>(a, kmap, vmap, work, box_shift);
}

// Joins the partial sums of the pairs that were cut, in CTA order, and
// writes the zero rows of sequences without positions.
constexpr int kFewGridMax = 512;          // CTAs, and so pieces of a pair
constexpr int kJoinThreads = 128;

template <typename T, int HD>
__global__ void __launch_bounds__(kJoinThreads)
    paged_few_join_kernel(const __grid_constant__ PagedAttnArgs a, FewWork work) {
  using S = Storage<T>;
  __shared__ float weight[kFewGridMax][kFewRows];
  __shared__ float inv[kFewRows];
  const int b = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int shift = ilog2(a.page_size);
  const int G = a.n_q_heads / a.n_kv_heads;
  const SeqView s = sequence_view(a, b, shift);
  if (s.bad && h == 0 && tid == 0 && a.status) atomicOr(a.status, VL_STATUS_BAD_PAGE);
  const int tiles = few_tiles(s);
  pdl_wait();
  T* out = static_cast<T*>(a.out) + static_cast<int64_t>(s.start) * a.out_row_stride +
           static_cast<int64_t>(h) * G * HD;
  if (tiles == 0) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const int64_t vecs = static_cast<int64_t>(s.rows) * G * (HD / 8);
    for (int64_t i = tid; i < vecs; i += kJoinThreads)
      st_vec(out + i / (G * (HD / 8)) * a.out_row_stride + i % (G * (HD / 8)) * 8, zero);
    return;
  }
  const int64_t share = work.base[a.batch + 1];
  const int64_t u0 = work.base[b] + static_cast<int64_t>(h) * tiles, u1 = u0 + tiles;
  const int64_t c0 = divide(u0, share), c1 = divide(u1 - 1, share);
  if (c0 == c1) return;                   // finished where it was computed
  const int pieces = static_cast<int>(c1 - c0) + 1, R = s.rows * G;
  // a CTA's first piece is its slot 0: only the pair's first may be the second
  const float* part = work.part + 2 * c0 * few_partial_floats(HD);
  const int late = u0 != c0 * share ? 1 : 0;
  auto slot = [&](int k) {
    return part + static_cast<int64_t>(2 * k + (k == 0 ? late : 0)) * few_partial_floats(HD);
  };
  // A thread's share of the first pieces is asked for before their weights are
  // known: the sums (four dims of a row) and, eight threads a row, (max, sum).
  constexpr int kTeam = kJoinThreads / kFewRows, kAhead = 8;
  const int n = tid / kTeam, k0 = tid % kTeam;
  float2 ml[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    ml[u] = make_float2(-INFINITY, 0.0f);
    if (n < R && k0 + u * kTeam < pieces)
      ml[u] = __ldcg(reinterpret_cast<const float2*>(slot(k0 + u * kTeam) + kFewRows * HD + 2 * n));
  }
  float4 x[kAhead];
  auto ask = [&](int i, int k) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (k + u < pieces && i < R * (HD / 4))
        x[u] = __ldcg(reinterpret_cast<const float4*>(slot(k + u)) + i);   // rows lie densely
  };
  ask(tid, 0);
  auto more = [&](int k) {                // (max, sum) of a piece behind the first 32
    return __ldcg(reinterpret_cast<const float2*>(slot(k) + kFewRows * HD + 2 * n));
  };
  float M = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), L = 0.0f;
  if (n < R)
    for (int k = k0 + 4 * kTeam; k < pieces; k += kTeam) M = fmaxf(M, more(k).x);
#pragma unroll
  for (int o = kTeam / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (n < R) {
    auto note = [&](int k, const float2& v) {
      const float w = v.x == -INFINITY ? 0.0f : exp2f(v.x - M);
      weight[k][n] = w;
      L = fmaf(v.y, w, L);
    };
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (k0 + u * kTeam < pieces) note(k0 + u * kTeam, ml[u]);
    for (int k = k0 + 4 * kTeam; k < pieces; k += kTeam) note(k, more(k));
  }
#pragma unroll
  for (int o = kTeam / 2; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  if (k0 == 0) inv[n] = L == 0.0f ? 0.0f : 1.0f / L;
  __syncthreads();
  for (int i = tid; i < R * (HD / 4); i += kJoinThreads) {
    const int row = i / (HD / 4), d = (i % (HD / 4)) * 4;
    float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < pieces; k += kAhead) {
      if (i != tid || k > 0) ask(i, k);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (k + u < pieces) {
          const float w = weight[k + u][row];
          f.x = fmaf(x[u].x, w, f.x);
          f.y = fmaf(x[u].y, w, f.y);
          f.z = fmaf(x[u].z, w, f.z);
          f.w = fmaf(x[u].w, w, f.w);
        }
    }
    const float r = inv[row];
    const uint2 y = make_uint2(pack16(f.x * r, f.y * r, T()), pack16(f.z * r, f.w * r, T()));
    *reinterpret_cast<uint2*>(out + static_cast<int64_t>(row / G) * a.out_row_stride +
                              static_cast<int64_t>(row % G) * HD + d) = y;
  }
}

// Few pairs and tables of at most 1024 positions: one launch of clusters,
// instead of the line and its join.  4 sequences of 500, G = 4: 6.7 us against
// 8.0 (4 tokens each 9.0 against 12.2); of 200: 5.6 against 7.6; of 1000: 8.1
// against 8.8; of 2000 the line is better, 9.6 against 10.9.  Clusters of eight
// gain 0.1 us at 500, lose 0.5 at 200, and fewer of them fit.
bool few_by_cluster(const PagedAttnArgs& a) {
  const int64_t pairs = static_cast<int64_t>(a.batch) * a.n_kv_heads;
  const int64_t tiles = (static_cast<int64_t>(a.max_pages) * a.page_size + kFewTile - 1) / kFewTile;
  return pairs * kFewCluster <= 2 * sm_count() && tiles <= 4 * kFewCluster;
}

int few_grid() {
  const int n = sm_count() * kFewCtasPerSm;
  return n < kFewGridMax ? n : kFewGridMax;
}

size_t few_workspace(int64_t batch, int hd) {
  return ((static_cast<size_t>(batch) + 2) * 8 + 255) / 256 * 256 +
         static_cast<size_t>(few_grid()) * 2 * few_partial_floats(hd) * sizeof(float);
}

template <typename T, int HD, int NT>
cudaError_t few_launch(const PagedAttnArgs& a, void* workspace, bool pdl, cudaStream_t stream) {
  FewWork work;
  work.base = static_cast<int64_t*>(workspace);
  work.part = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                       ((static_cast<size_t>(a.batch) + 2) * 8 + 255) / 256 * 256);
  const int box = a.page_size < kFewTile ? a.page_size : kFewTile;
  int box_shift = 0;
  while ((1 << box_shift) < box) ++box_shift;
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap kmap, vmap;
  if (!encode_cache_map(&kmap, a.k_cache, bf16, HD, a.n_kv_heads, a.page_size, a.num_pages,
                        a.page_stride, box) ||
      !encode_cache_map(&vmap, a.v_cache, bf16, HD, a.n_kv_heads, a.page_size, a.num_pages,
                        a.page_stride, box))
    return cudaErrorNotSupported;
  constexpr size_t smem = 1024 + static_cast<size_t>(kFewStages) * 2 * kFewTile * HD * sizeof(T) +
                          sizeof(FewSmem<T, HD, NT>);
  auto kernel = paged_few_kernel<T, HD, NT>;
  auto by_cluster = paged_few_cluster_kernel<T, HD, NT, kFewCluster>;
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem));
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(by_cluster, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  if (few_by_cluster(a))
    return launch_kernel(by_cluster,
                         dim3(static_cast<unsigned>(a.batch * a.n_kv_heads * kFewCluster)),
                         dim3(kFewThreads), smem, stream, pdl, a, kmap, vmap, work, box_shift);
  e = launch_kernel(kernel, dim3(static_cast<unsigned>(few_grid())), dim3(kFewThreads), smem,
                    stream, pdl, a, kmap, vmap, work, box_shift);
  if (e != cudaSuccess) return e;
  return launch_kernel(paged_few_join_kernel<T, HD>,
                       dim3(static_cast<unsigned>(a.batch), static_cast<unsigned>(a.n_kv_heads)),
                       dim3(kJoinThreads), 0, stream, true, a, work);
}

template <typename T>
cudaError_t few_typed(const PagedAttnArgs& a, void* workspace, bool pdl, cudaStream_t stream) {
  const int rows = a.max_q_len * (a.n_q_heads / a.n_kv_heads);
  if (a.head_dim == 128)
    return rows <= 8 ? few_launch<T, 128, 1>(a, workspace, pdl, stream)
                     : few_launch<T, 128, 2>(a, workspace, pdl, stream);
  return rows <= 8 ? few_launch<T, 64, 1>(a, workspace, pdl, stream)
                   : few_launch<T, 64, 2>(a, workspace, pdl, stream);
}

// ---------------------------------------------------------------------------
// any type and head_dim
// ---------------------------------------------------------------------------
// A warp per (token, query head): a lane takes one of 32 positions for the
// scores, then every 32nd dim for the sums.  For f32 and head dims without
// a tensor-core kernel: right everywhere, not fast.
constexpr int kAnyWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kAnyWarps * 32)
    paged_any_kernel(const __grid_constant__ PagedAttnArgs a) {
  using S = Storage<T>;
  constexpr int E = S::kVec;
  __shared__ float qs[kAnyWarps][256];
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.y * kAnyWarps + warp;
  const int shift = ilog2(a.page_size), mask = a.page_size - 1;
  pdl_wait();
  pdl_release();
  const int b = find_sequence(a.q_start, a.batch, t, lane);
  const SeqView s = sequence_view(a, b, shift);
  if (s.bad && head == 0 && lane == 0 && a.status) atomicOr(a.status, VL_STATUS_BAD_PAGE);
  if (head >= a.n_q_heads || t < s.start || t >= s.start + static_cast<int64_t>(s.rows)) return;
  const int hd = a.head_dim, kvh = head / (a.n_q_heads / a.n_kv_heads);
  const int64_t row = static_cast<int64_t>(a.n_kv_heads) * hd;
  const T* qrow = static_cast<const T*>(a.q) + t * a.q_row_stride + static_cast<int64_t>(head) * hd;
  for (int d = lane; d < hd; d += 32) qs[warp][d] = S::to_float(qrow[d]);
  __syncwarp();
  const int len = s.len > 0 ? s.len - s.rows + static_cast<int>(t - s.start) + 1 : 0;
  float m = -INFINITY, l = 0.0f, o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = 0.0f;
  for (int p0 = 0; p0 < len; p0 += 32) {
    const int p = p0 + lane;
    int64_t at = -1;                      // element offset of the position's row, -1: zeros
    float sc = -INFINITY;
    if (p < len) {
      const int page = a.page_table[b * a.table_stride + (p >> shift)];
      if (page >= 0 && page < a.num_pages) {
        at = page * a.page_stride + (p & mask) * row + static_cast<int64_t>(kvh) * hd;
      } else if (a.status) {
        atomicOr(a.status, VL_STATUS_BAD_PAGE);
      }
      float dot = 0.0f;
      if (at >= 0) {
        const T* krow = static_cast<const T*>(a.k_cache) + at;
        for (int d = 0; d < hd; d += E) {
          float f[E];
          S::unpack(ld_vec(krow + d), f);
#pragma unroll
          for (int e = 0; e < E; ++e) dot = fmaf(f[e], qs[warp][d + e], dot);
        }
      }
      sc = dot * a.scale * kLog2e;
    }
    const float m_new = fmaxf(m, warp_max(sc));
    const float alpha = m_new == -INFINITY ? 1.0f : exp2f(m - m_new);
    const float w = sc == -INFINITY ? 0.0f : exp2f(sc - m_new);
    m = m_new;
    l = fmaf(l, alpha, warp_sum(w));
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= alpha;
    const int n = min(32, len - p0);
    for (int j = 0; j < n; ++j) {
      const float wj = __shfl_sync(0xffffffffu, w, j);
      const int64_t aj = __shfl_sync(0xffffffffu, at, j);
      if (aj < 0) continue;
      const T* vrow = static_cast<const T*>(a.v_cache) + aj;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i * 32 < hd) o[i] = fmaf(wj, S::to_float(vrow[i * 32 + lane]), o[i]);
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(a.out) + t * a.out_row_stride + static_cast<int64_t>(head) * hd;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i * 32 < hd) out[i * 32 + lane] = S::from_float(o[i] * inv);
}

template <typename T>
cudaError_t any_launch(const PagedAttnArgs& a, bool pdl, cudaStream_t stream) {
  return launch_kernel(paged_any_kernel<T>,
                       dim3(static_cast<unsigned>(a.tokens),
                            static_cast<unsigned>((a.n_q_heads + kAnyWarps - 1) / kAnyWarps)),
                       dim3(kAnyWarps * 32), 0, stream, pdl, a);
}

enum class Kind { kFew, kChunk, kAny };

// Up to 16 rows per kv head (two 8-wide MMA columns) the few-token kernel
// streams the cache; from there on the tcgen05 kernel's 128-row blocks re-read
// it less often.  64 x 4 tokens over 2048 positions, G = 4 (16 rows): 57.6
// us against 71.4; 16 x 4 over 1000: 16.8 against 29.0; 4 x 1 over 500: 6.7
// against 16.2.
Kind paged_kind(int64_t max_q_len, int n_q_heads, int n_kv_heads, int head_dim, int dtype) {
  if (dtype == kDtypeF32 || (head_dim != 64 && head_dim != 128)) return Kind::kAny;
  return max_q_len * (n_q_heads / n_kv_heads) <= kFewRows ? Kind::kFew : Kind::kChunk;
}

}  // namespace

bool encode_cache_map(CUtensorMap* map, const void* cache, bool bf16, int head_dim,
                      int n_kv_heads, int page_size, int64_t num_pages, int64_t page_stride,
                      int box_rows) {
  EncodeTiled encode = encoder();
  if (encode == nullptr) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim),
                              static_cast<cuuint64_t>(n_kv_heads),
                              static_cast<cuuint64_t>(page_size),
                              static_cast<cuuint64_t>(num_pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(head_dim) * 2,
                                 static_cast<cuuint64_t>(head_dim) * n_kv_heads * 2,
                                 static_cast<cuuint64_t>(page_stride) * 2};
  const cuuint32_t box[4] = {64, 1, static_cast<cuuint32_t>(box_rows), 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                const_cast<void*>(cache), dims, strides, box, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool encode_rows_map(CUtensorMap* map, const void* rows, bool bf16, int head_dim, int n_heads,
                     int64_t tokens, int64_t row_stride, int box_heads, int box_tokens) {
  EncodeTiled encode = encoder();
  if (encode == nullptr) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(n_heads),
                              static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_dim) * 2,
                                 static_cast<cuuint64_t>(row_stride) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads),
                             static_cast<cuuint32_t>(box_tokens)};
  const cuuint32_t estr[3] = {1, 1, 1};
  return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                const_cast<void*>(rows), dims, strides, box, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

size_t paged_attention_workspace_bytes(int64_t batch, int64_t max_q_len, int n_q_heads,
                                       int n_kv_heads, int head_dim, int dtype) {
  switch (paged_kind(max_q_len, n_q_heads, n_kv_heads, head_dim, dtype)) {
    case Kind::kFew: return few_workspace(batch, head_dim);
    case Kind::kChunk: return paged_attention_tc_workspace_bytes(head_dim);
    default: return 16;
  }
}

cudaError_t launch_paged_attention(const PagedAttnArgs& a, int dtype, void* workspace, bool pdl,
                                   cudaStream_t stream) {
  if (a.batch == 0 || a.tokens == 0) return cudaSuccess;
  switch (paged_kind(a.max_q_len, a.n_q_heads, a.n_kv_heads, a.head_dim, dtype)) {
    case Kind::kFew:
      return dtype == kDtypeBF16 ? few_typed<__nv_bfloat16>(a, workspace, pdl, stream)
                                 : few_typed<__half>(a, workspace, pdl, stream);
    case Kind::kChunk: return launch_paged_attention_tc(a, dtype, workspace, pdl, stream);
    default:
      if (dtype == kDtypeF32) return any_launch<float>(a, pdl, stream);
      return dtype == kDtypeF16 ? any_launch<__half>(a, pdl, stream)
                                : any_launch<__nv_bfloat16>(a, pdl, stream);
  }
}

}  // namespace vl
