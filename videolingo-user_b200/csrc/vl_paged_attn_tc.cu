// Attention of a chunk of new tokens over a paged KV cache on the sm_100a
// tensor cores (tcgen05 + TMA + TMEM).
//
//   S = scale Q K^T (causal),  P = exp2(log2e S - m),  O = P V / sum P
//
// Bound by the tensor cores and, as closely, by exp2: a 128 x 128 tile of S
// costs 512 cycles of MMA for each of its two products at head_dim 128 and
// 1024 cycles of the 16-per-cycle exponential unit.  So the two must run
// side by side:
//   * a CTA takes 256 query rows of one kv head as two blocks of 128 and
//     works on both against the same K and V tiles of 128 positions.  While
//     the tensor cores run one block's P V and next Q K^T, the other block's
//     four warps take their exponentials;
//   * a row of the tile is one thread's: S comes from tensor memory
//     (tcgen05.ld, lane = row), maximum and sum need no shuffles, P goes
//     back as 16-bit over the same columns and is the A operand of P V from
//     there;
//   * query rows are (token, query head of the group) pairs, so the G heads
//     that share a kv head share its tiles, and a TMA box of [tokens][G][64]
//     brings them in that order;
//   * O stays in tensor memory.  It is rescaled only when a row's maximum
//     has grown by more than 2^8 since the last time: until then weights are
//     taken about the old maximum, which fp32 sums and both 16-bit types
//     hold (P <= 2^8).
//   * one warp turns page ids into TMA boxes, one thread issues the MMAs.
//     CTAs are persistent; the next item's Q and K arrive while the last one
//     is being finished.
// Items (256 rows x kv head) are dealt heaviest first.  When there are fewer
// than SMs, the positions of each are cut into pieces whose partial sums a
// second launch joins.
#include <cuda.h>

#include <atomic>
#include <cmath>

#include "vl_common.cuh"
#include "vl_kernels.h"
#include "vl_paged.cuh"
#include "vl_tma.cuh"

namespace vl {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 128;                // rows of a block (MMA M)
constexpr int kTile = 128;                // positions of a tile
constexpr int kStages = 2;                // of K and of V
constexpr int kSoftThreads = 256;         // two blocks' warps
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr int kThreads = 320;
constexpr float kRescaleLog2 = 8.0f;

template <int HD>
struct Shape {
  static constexpr int kHalves = HD / 64;
  static constexpr int kColumn = kRows * 128;          // bytes: 128 rows x 64 dims
  static constexpr int kMatrix = kHalves * kColumn;    // 128 rows x HD
  static constexpr int kQ = 0;                         // two blocks
  static constexpr int kK = 2 * kMatrix;
  static constexpr int kV = kK + kStages * kMatrix;
  static constexpr int kBars = kV + kStages * kMatrix;
  static constexpr int kBytes = kBars + 256 + 1024;    // barriers, and the ring's alignment
};

struct Bars {
  uint64_t q_full, q_empty;
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], p_half[2], p_ready[2], o_done[2];
  uint64_t end;
  uint32_t tmem;
  int bad;
};
static_assert(sizeof(Bars) <= 256, "barrier block");

struct TcWork {
  float* part;        // split: [cell * splits + s][256 rows][HD], then [..][256] (max, sum)
  float2* ml;
  int splits;
  int tiles;          // q tiles of a sequence, at most
  int cells;          // tiles * batch * kv heads
};

// One piece of work: a block pair of a sequence and kv head, and a run of
// position tiles.
struct Piece {
  int b, h;
  SeqView s;
  int tok0;           // first token of the pair
  int j0;             // first position tile
  int count[2];       // tiles of each block
  int rows_tok;       // tokens of a block
  int tiles;          // block pairs of the sequence
  int k;              // this one, from the sequence's end
  bool lead;          // the sequence's first piece
};

__device__ __forceinline__ Piece piece_of(const PagedAttnArgs& a, const TcWork& w, int index,
                                          int shift, int group) {
  Piece p;
  const int cell = index / w.splits, split = index - cell * w.splits;
  const int per = a.batch * a.n_kv_heads;
  const int rest = cell % per;
  p.k = cell / per;
  p.b = rest / a.n_kv_heads;
  p.h = rest - p.b * a.n_kv_heads;
  p.rows_tok = kRows / group;
  p.s = sequence_view(a, p.b, shift);
  const int pair = 2 * p.rows_tok;
  p.tiles = (p.s.rows + pair - 1) / pair;
  p.tok0 = (p.tiles - 1 - p.k) * pair;
  p.lead = p.k == 0 && p.h == 0 && split == 0;
  int n[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int first = p.tok0 + i * p.rows_tok;
    const int last = min(p.s.rows, first + p.rows_tok);
    const int see = p.s.len - p.s.rows + last;         // positions of the block's last token
    n[i] = p.k < p.tiles && first < p.s.rows && see > 0 && p.s.len > 0 ? (see + kTile - 1) / kTile : 0;
  }
  const int all = max(n[0], n[1]);
  p.j0 = static_cast<int>(static_cast<int64_t>(all) * split / w.splits);
  const int j1 = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / w.splits);
#pragma unroll
  for (int i = 0; i < 2; ++i) p.count[i] = max(0, min(j1, n[i]) - p.j0);
  return p;
}

__device__ __forceinline__ bool wait_or_bad(uint64_t* bar, uint32_t parity, int* bad) {
  for (uint32_t i = 0; i < (1u << 22); ++i) {
    if (mbarrier_test(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(bad)) return false;
  }
  atomicExch(bad, 1);
  return false;
}

__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_addr(bar))
               : "memory");
}

// Shared-memory descriptors in the 128-byte swizzle.  K-major (Q, K): 8-row
// groups 1 KB apart.  MN-major (V as B: positions are its K, 64 dims lie
// contiguous): 8-position groups 1 KB apart, the next 64 dims a column on.
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t leading, uint32_t stride) {
  return static_cast<uint64_t>((addr >> 4) & 0x3fff) |
         (static_cast<uint64_t>(leading >> 4) << 16) | (static_cast<uint64_t>(stride >> 4) << 32) |
         (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
template <typename T>
__device__ constexpr uint32_t instruction(int n, bool b_mn_major) {
  return (1u << 4) | ((std::is_same<T, __nv_bfloat16>::value ? 1u : 0u) << 7) |
         ((std::is_same<T, __nv_bfloat16>::value ? 1u : 0u) << 10) |
         ((b_mn_major ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 32 columns of this thread's lane.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
// Loads issued so far have arrived; ties the registers to the wait, so that
// no use of them moves above it.
template <int N>
__device__ __forceinline__ void tmem_tie(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
template <int N>
__device__ __forceinline__ void tmem_load_wait(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  tmem_tie<N>(r);
}
// Scores from `seen` on become -inf.
template <int N>
__device__ __forceinline__ void hide(uint32_t* r, int seen) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i >= seen) r[i] = 0xff800000u;
}
__device__ __forceinline__ void tmem_store_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(uint32_t a, uint32_t b, uint32_t c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;"
      : "=f"(y)
      : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
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
__device__ __forceinline__ uint32_t pack16(float lo, float hi, __nv_bfloat16) {
  return pack_bf16x2(lo, hi);
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, __half) {
  return pack_f16x2(lo, hi);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
    paged_chunk_kernel(const __grid_constant__ PagedAttnArgs a,
                       const __grid_constant__ CUtensorMap qmap,
                       const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, TcWork w, int box_shift) {
  using S = Storage<T>;
  using L = Shape<HD>;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw0 = smem_addr(smem_raw);
  const uint32_t base = (raw0 + 1023) & ~1023u;
  Bars& bars = *reinterpret_cast<Bars*>(smem_raw + (base - raw0) + L::kBars);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int shift = ilog2(a.page_size);
  const int G = a.n_q_heads / a.n_kv_heads;
  const int pieces = w.cells * w.splits;

  if (tid == 0) {
    mbarrier_init(&bars.q_full, 1);
    mbarrier_init(&bars.q_empty, 1);
    for (int s = 0; s < kStages; ++s) {
      mbarrier_init(&bars.k_full[s], 1);
      mbarrier_init(&bars.k_empty[s], 1);
      mbarrier_init(&bars.v_full[s], 1);
      mbarrier_init(&bars.v_empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbarrier_init(&bars.s_full[i], 1);
      mbarrier_init(&bars.p_half[i], kSoftThreads / 64);    // a block's warps
      mbarrier_init(&bars.p_ready[i], kSoftThreads / 64);
      mbarrier_init(&bars.o_done[i], 1);
    }
    mbarrier_init(&bars.end, 1);
    bars.bad = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&bars.tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = bars.tmem;
  pdl_wait();
  pdl_release();

  if (warp == kProducerWarp) {
    // ---- copies: Q of a piece, then its K and V tiles in turn ----
    const int box_rows = 1 << box_shift;
    uint32_t tile = 0, item = 0;          // tiles and pieces so far
    bool ok = true;
    for (int index = blockIdx.x; ok && index < pieces; index += gridDim.x) {
      const Piece p = piece_of(a, w, index, shift, G);
      const int n = max(p.count[0], p.count[1]);
      if (n == 0) continue;
      if (item > 0 && !wait_or_bad(&bars.q_empty, (item - 1) & 1, &bars.bad)) break;
      if (elect_lane()) {
        const uint32_t bytes = L::kHalves * 128 * G * p.rows_tok;
        mbarrier_expect(&bars.q_full, bytes * ((p.count[0] > 0) + (p.count[1] > 0)));
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (p.count[i] > 0)
#pragma unroll
            for (int c = 0; c < L::kHalves; ++c)
              tma_load_3d(base + L::kQ + i * L::kMatrix + c * L::kColumn, &qmap, c * 64, p.h * G,
                          p.s.start + p.tok0 + i * p.rows_tok, &bars.q_full);
      }
      __syncwarp();
      ++item;
      for (int jj = 0; jj < n; ++jj, ++tile) {
        const int pos0 = (p.j0 + jj) * kTile;
        const int need = (min(kTile, p.s.len - pos0) + box_rows - 1) >> box_shift;
        // lane l looks up the l-th box's page, all before the waits
        int page = 0;
        if (lane < need) {
          page = a.page_table[p.b * a.table_stride + ((pos0 + (lane << box_shift)) >> shift)];
          if (page < 0 || page >= a.num_pages) {       // read as rows of zeros
            page = static_cast<int>(a.num_pages);
            if (a.status) atomicOr(a.status, VL_STATUS_BAD_PAGE);
          }
        }
        const int st = tile % kStages;
        const uint32_t parity = ((tile / kStages) & 1) ^ 1;
        const uint32_t bytes = static_cast<uint32_t>(need) * box_rows * 128 * L::kHalves;
        auto fetch = [&](uint32_t matrix, const CUtensorMap* map, uint64_t* full) {
          if (elect_lane()) mbarrier_expect(full, bytes);
          __syncwarp();
          for (int j = 0; j < need; ++j) {
            const int pj = __shfl_sync(0xffffffffu, page, j);
            const uint32_t dst = matrix + st * L::kMatrix + j * box_rows * 128;
            const int row = (pos0 + (j << box_shift)) & (a.page_size - 1);
            if (elect_lane()) {
#pragma unroll
              for (int c = 0; c < L::kHalves; ++c)
                tma_load_4d(dst + c * L::kColumn, map, c * 64, p.h, row, pj, full);
            }
            __syncwarp();
          }
        };
        if (tile >= kStages && !wait_or_bad(&bars.k_empty[st], parity, &bars.bad)) {
          ok = false;
          break;
        }
        fetch(base + L::kK, &kmap, &bars.k_full[st]);
        if (tile >= kStages && !wait_or_bad(&bars.v_empty[st], parity, &bars.bad)) {
          ok = false;
          break;
        }
        fetch(base + L::kV, &vmap, &bars.v_full[st]);
      }
    }
    if (*reinterpret_cast<volatile int*>(&bars.bad)) {
      // leave no copy in flight (each wait is bounded; what was never asked
      // for lets them run out)
      if (item > 0) (void)mbarrier_wait(&bars.q_full, (item - 1) & 1);
      for (uint32_t t = tile < kStages ? 0 : tile - kStages; t <= tile; ++t) {
        const uint32_t parity = (t / kStages) & 1;
        for (int i = 0; i < 1000 && !mbarrier_test(&bars.k_full[t % kStages], parity); ++i) {}
        for (int i = 0; i < 1000 && !mbarrier_test(&bars.v_full[t % kStages], parity); ++i) {}
      }
    }
  } else if (warp == kMmaWarp) {
    // ---- products: the warp waits, an elected lane issues ----
    constexpr uint32_t kIdescS = instruction<T>(kTile, false);
    constexpr uint32_t kIdescO = instruction<T>(HD, true);
    uint32_t tile = 0, item = 0, used[2] = {0, 0};
    auto scores = [&](int i, int st) {                 // S_i = Q_i K^T
      const uint32_t q = base + L::kQ + i * L::kMatrix, k = base + L::kK + st * L::kMatrix;
      if (elect_lane()) {
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = (kk >> 2) * L::kColumn + (kk & 3) * 32;
          mma_ss(tmem + i * kTile, desc(q + off, 16, 1024), desc(k + off, 16, 1024), kIdescS,
                 kk > 0);
        }
        commit(&bars.s_full[i]);
      }
      __syncwarp();
    };
    // O_i (+)= P_i V over one half of the tile's positions
    auto values = [&](int i, int st, int half, bool first) {
      const uint32_t v = base + L::kV + st * L::kMatrix + half * (kTile / 2) * 128;
      const uint32_t p = tmem + i * kTile + kTile / 2 + half * (kTile / 4);
      if (elect_lane()) {
#pragma unroll
        for (int kk = 0; kk < kTile / 32; ++kk)
          mma_ts(tmem + 2 * kTile + i * HD, p + kk * 8, desc(v + kk * 2048, L::kColumn, 1024),
                 kIdescO, !first || kk > 0);
      }
      __syncwarp();
    };
    auto signal = [&](uint64_t* bar) {                 // when the products so far are done
      if (elect_lane()) commit(bar);
      __syncwarp();
    };
    bool ok = true;
    for (int index = blockIdx.x; ok && index < pieces; index += gridDim.x) {
      const Piece p = piece_of(a, w, index, shift, G);
      const int n = max(p.count[0], p.count[1]);
      if (n == 0) continue;
      ok = wait_or_bad(&bars.q_full, item & 1, &bars.bad) &&
           wait_or_bad(&bars.k_full[tile % kStages], (tile / kStages) & 1, &bars.bad);
      if (!ok) break;
      fence_after();
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (p.count[i] > 0) scores(i, tile % kStages);
      signal(&bars.k_empty[tile % kStages]);
      if (n == 1) signal(&bars.q_empty);
      for (int jj = 0; ok && jj < n; ++jj, ++tile) {
        const int st = tile % kStages;
        const uint32_t next = tile + 1;
        ok = wait_or_bad(&bars.v_full[st], (tile / kStages) & 1, &bars.bad);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (ok && jj < p.count[i]) {
            ok = wait_or_bad(&bars.p_half[i], used[i] & 1, &bars.bad);
            if (ok) {
              fence_after();
              values(i, st, 1, jj == 0);
              ok = wait_or_bad(&bars.p_ready[i], used[i] & 1, &bars.bad);
            }
            if (ok) {
              ++used[i];
              fence_after();
              values(i, st, 0, false);
              if (jj + 1 == p.count[i]) signal(&bars.o_done[i]);
            }
          }
          if (ok && jj + 1 < p.count[i]) {
            ok = wait_or_bad(&bars.k_full[next % kStages], (next / kStages) & 1, &bars.bad);
            if (ok) {
              fence_after();
              scores(i, next % kStages);
            }
          }
        }
        if (!ok) break;
        signal(&bars.v_empty[st]);
        if (jj + 1 < n) {
          signal(&bars.k_empty[next % kStages]);
          if (jj + 2 == n) signal(&bars.q_empty);
        }
      }
      ++item;
    }
    // every MMA has ended, and with it the arrivals that it owes
    signal(&bars.end);
    (void)mbarrier_wait(&bars.end, 0);
  } else if (warp < kProducerWarp) {
    // ---- softmax: a thread per row ----
    const int i = warp >> 2;                           // block
    const int r = tid & (kRows - 1);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + i * kTile + lanes, to = tmem + 2 * kTile + i * HD + lanes;
    const float scale = a.scale * kLog2e;
    uint32_t tile = 0, used = 0, finished = 0;
    bool ok = true;
    for (int index = blockIdx.x; ok && index < pieces; index += gridDim.x) {
      const Piece p = piece_of(a, w, index, shift, G);
      if (p.lead && p.s.bad && tid == 0 && a.status) atomicOr(a.status, VL_STATUS_BAD_PAGE);
      if (p.s.len == 0) {                 // nothing cached, or bad lengths: zero rows
        if (index % w.splits != 0 || r >= G * p.rows_tok) continue;
        for (int64_t t = static_cast<int64_t>(p.k) * 2 * p.rows_tok + i * p.rows_tok + r / G;
             t < p.s.rows; t += static_cast<int64_t>(w.tiles) * 2 * p.rows_tok) {
          T* out = static_cast<T*>(a.out) + (p.s.start + t) * a.out_row_stride +
                   static_cast<int64_t>(p.h * G + r % G) * HD;
          for (int c = 0; c < HD; c += 8) st_vec(out + c, make_uint4(0, 0, 0, 0));
        }
        continue;
      }
      if (p.k >= p.tiles) continue;
      const int tok = p.tok0 + i * p.rows_tok + r / G, g = r % G;
      const bool mine = r < G * p.rows_tok && tok < p.s.rows;
      const int see = mine ? p.s.len - p.s.rows + tok + 1 : 0;
      float m = -INFINITY, l = 0.0f;
      for (int jj = 0; jj < p.count[i]; ++jj) {
        if (!(ok = wait_or_bad(&bars.s_full[i], used & 1, &bars.bad))) break;
        ++used;
        fence_after();
        const int pos0 = (p.j0 + jj) * kTile;
        // The row in two halves.  P takes the columns of the upper one, so
        // that the lower can wait in tensor memory while the upper's
        // exponentials are taken: a thread then holds 64 to 96 scores, not
        // 128 and what it makes of them.
        uint32_t lo[kTile / 2], hi[kTile / 2];
        tmem_load32(ts, lo);
        tmem_load32(ts + 32, lo + 32);
        tmem_load32(ts + 64, hi);
        tmem_load32(ts + 96, hi + 32);
        tmem_load_wait<kTile / 2>(lo);
        tmem_tie<kTile / 2>(hi);
        const bool cut = pos0 + kTile > see;
        if (cut) {
          hide<kTile / 2>(lo, see - pos0);
          hide<kTile / 2>(hi, see - pos0 - kTile / 2);
        }
        float mx = max3(lo[0], hi[0], lo[1]), my = max3(lo[2], hi[2], hi[1]);
#pragma unroll
        for (int c = 3; c + 1 < kTile / 2; c += 2) {
          mx = max3(__float_as_uint(mx), lo[c], lo[c + 1]);
          my = max3(__float_as_uint(my), hi[c], hi[c + 1]);
        }
        mx = max3(__float_as_uint(mx), lo[kTile / 2 - 1], hi[kTile / 2 - 1]);
        mx = fmaxf(mx, my);
        mx *= scale;
        if (__any_sync(0xffffffffu, mx > m + kRescaleLog2)) {
          const float m_new = fmaxf(m, mx);
          const float f = m_new == -INFINITY ? 1.0f : ex2(m - m_new);
          l *= f;
          m = m_new;
          if (jj > 0) {
            // the products that wrote O are done: this tile's scores were
            // issued behind them
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
              uint32_t o[32];
              tmem_load32(to + c, o);
              tmem_load_wait<32>(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_store32(to + c, o);
            }
          }
        }
        if (pos0 + kTile > p.s.len) {
          // rows of V past the end hold anything: their weights are 0, and so
          // must they be
          const uint32_t t = tile + jj;
          if (!(ok = wait_or_bad(&bars.v_full[t % kStages], (t / kStages) & 1, &bars.bad))) break;
          const uint32_t v = base + L::kV + (t % kStages) * L::kMatrix;
          const int past = p.s.len - pos0;
          for (int z = r; z < (kTile - past) * (HD / 8); z += kRows) {
            const int row = past + z / (HD / 8), ch = z % (HD / 8);
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(
                             v + (ch >> 3) * L::kColumn + row * 128 + (((ch & 7) ^ (row & 7)) << 4)),
                         "r"(0)
                         : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        const float off = m == -INFINITY ? 0.0f : -m;
        const uint64_t scale2 = pair_of(scale, scale), off2 = pair_of(off, off);
        // P rounds to the storage type, as its tensor-core operand: half a
        // step per weight, against a sum that stays in fp32
        uint64_t sum[2] = {0, 0};
        auto weights = [&](const uint32_t* x, int part) {   // 32 positions of the tile
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 z = halves_of(fma2(pair_of(x[e], x[e + 1]), scale2, off2));
            const float e0 = ex2(z.x), e1 = ex2(z.y);
            sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pair_of(e0, e1));
            pk[e / 2] = pack16(e0, e1, T());
          }
          tmem_store16(ts + kTile / 2 + part * 16, pk);
        };
        auto publish = [&](uint64_t* bar) {                 // products over them may start
          tmem_store_wait();
          fence_before();
          __syncwarp();
          if (lane == 0) mbarrier_arrive(bar);
        };
        tmem_load32(ts, lo);
        weights(hi, 2);
        weights(hi + 32, 3);
        tmem_load_wait<32>(lo);
        publish(&bars.p_half[i]);
        tmem_load32(ts + 32, lo + 32);
        if (cut) hide<32>(lo, see - pos0);
        weights(lo, 0);
        tmem_load_wait<32>(lo + 32);
        if (cut) hide<32>(lo + 32, see - pos0 - 32);
        weights(lo + 32, 1);
        publish(&bars.p_ready[i]);
        const float2 s0 = halves_of(add2(sum[0], sum[1]));
        l += s0.x + s0.y;
      }
      tile += max(p.count[0], p.count[1]);
      if (!ok) break;
      // ---- the piece's rows ----
      float inv = 0.0f;
      if (p.count[i] > 0) {
        if (!(ok = wait_or_bad(&bars.o_done[i], finished & 1, &bars.bad))) break;
        ++finished;
        fence_after();
        inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
      }
      const int64_t row256 = static_cast<int64_t>(index) * 2 * kRows + i * kRows + r;
      if (w.splits > 1 && p.count[i] > 0) {
        if (mine) w.ml[row256] = make_float2(m, l);
        inv = 1.0f;
      }
      T* out = static_cast<T*>(a.out) + static_cast<int64_t>(p.s.start + tok) * a.out_row_stride +
               static_cast<int64_t>(p.h * G + g) * HD;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        uint32_t o[32];
        if (p.count[i] > 0) {
          tmem_load32(to + c, o);
          tmem_load_wait<32>(o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (!mine) continue;
        if (w.splits > 1) {
          if (p.count[i] > 0) {
            float4* dst = reinterpret_cast<float4*>(w.part + row256 * HD + c);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              dst[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                   __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
          }
        } else {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              f[e] = inv == 0.0f ? 0.0f : __uint_as_float(o[8 * v + e]) * inv;
            st_vec(out + c + v * 8, S::pack(f));
          }
        }
      }
      fence_before();
    }
    if (!ok && r == 0 && a.status) atomicOr(a.status, VL_STATUS_TIMEOUT);
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                 : "memory");
  }
}

// Joins the sums of a cell's pieces, in order: one warp per row.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
    paged_chunk_join_kernel(const __grid_constant__ PagedAttnArgs a, TcWork w) {
  using S = Storage<T>;
  const int cell = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int shift = ilog2(a.page_size), G = a.n_q_heads / a.n_kv_heads;
  pdl_wait();
  constexpr int E = HD / 32;
  for (int rr = blockIdx.y * 8 + warp; rr < 2 * kRows; rr += gridDim.y * 8) {
    const int i = rr / kRows, r = rr % kRows;
    float M = -INFINITY, lsum = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    Piece p;
    for (int s = 0; s < w.splits; ++s) {
      p = piece_of(a, w, cell * w.splits + s, shift, G);
      if (p.k >= p.tiles || p.s.len == 0) return;
      if (p.count[i] == 0) continue;
      const int64_t row = (static_cast<int64_t>(cell) * w.splits + s) * 2 * kRows + rr;
      const float2 ml = w.ml[row];
      const float m_new = fmaxf(M, ml.x);
      const float f0 = M == -INFINITY ? 0.0f : exp2f(M - m_new);
      const float f1 = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - m_new);
      M = m_new;
      lsum = lsum * f0 + ml.y * f1;
      const float* src = w.part + row * HD + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * f0 + (f1 == 0.0f ? 0.0f : src[e] * f1);
    }
    const int tok = p.tok0 + i * p.rows_tok + r / G, g = r % G;
    if (r >= G * p.rows_tok || tok >= p.s.rows) continue;
    const float inv = lsum > 0.0f || lsum != lsum ? 1.0f / lsum : 0.0f;
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(p.s.start + tok) * a.out_row_stride +
             static_cast<int64_t>(p.h * G + g) * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = S::from_float(o[e] * inv);
  }
}

TcWork plan(int64_t tokens, int64_t batch, int64_t max_q_len, int n_q_heads, int n_kv_heads,
            int64_t max_positions) {
  TcWork w{};
  const int64_t pair = 2 * (kRows / (n_q_heads / n_kv_heads));
  const int64_t tiles = (max_q_len + pair - 1) / pair;
  w.tiles = static_cast<int>(tiles);
  const int64_t cells = tiles * batch * n_kv_heads;
  w.cells = cells > 0x3fffffff ? 0 : static_cast<int>(cells);   // the loops count in ints
  // cells that can hold rows
  int64_t live = tokens / pair + batch;
  if (live > tiles * batch) live = tiles * batch;
  live *= n_kv_heads;
  int64_t splits = sm_count() / (live > 0 ? live : 1);
  const int64_t most = max_positions / (4 * kTile);    // four tiles a piece, at least
  if (splits > most) splits = most;
  w.splits = splits < 1 ? 1 : static_cast<int>(splits);
  return w;
}

template <typename T, int HD>
cudaError_t chunk_launch(const PagedAttnArgs& a, void* workspace, bool pdl, cudaStream_t stream) {
  const int G = a.n_q_heads / a.n_kv_heads;
  const int64_t max_q_len = a.max_q_len < a.tokens ? a.max_q_len : a.tokens;
  TcWork w = plan(a.tokens, a.batch, max_q_len, a.n_q_heads, a.n_kv_heads,
                  static_cast<int64_t>(a.max_pages) * a.page_size);
  const int64_t rows = static_cast<int64_t>(w.cells) * w.splits * 2 * kRows;
  w.ml = static_cast<float2*>(workspace);
  w.part = reinterpret_cast<float*>(w.ml + rows);
  const int box = a.page_size < kTile ? a.page_size : kTile;
  int box_shift = 0;
  while ((1 << box_shift) < box) ++box_shift;
  const bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap qmap, kmap, vmap;
  if (!encode_rows_map(&qmap, a.q, bf16, HD, a.n_q_heads, a.tokens, a.q_row_stride, G, kRows / G) ||
      !encode_cache_map(&kmap, a.k_cache, bf16, HD, a.n_kv_heads, a.page_size, a.num_pages,
                        a.page_stride, box) ||
      !encode_cache_map(&vmap, a.v_cache, bf16, HD, a.n_kv_heads, a.page_size, a.num_pages,
                        a.page_stride, box))
    return cudaErrorNotSupported;
  auto kernel = paged_chunk_kernel<T, HD>;
  constexpr int smem = Shape<HD>::kBytes;
  static_assert(smem <= 227 * 1024, "chunk attention shared memory");
  static std::atomic<bool> configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  const int pieces = w.cells * w.splits;
  const int grid = pieces < sm_count() ? pieces : sm_count();
  e = launch_kernel(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem, stream, pdl, a,
                    qmap, kmap, vmap, w, box_shift);
  if (e != cudaSuccess || w.splits == 1) return e;
  return launch_kernel(paged_chunk_join_kernel<T, HD>,
                       dim3(static_cast<unsigned>(w.cells), 8), dim3(256), 0, stream, true, a, w);
}

}  // namespace

size_t paged_attention_tc_workspace_bytes(int64_t tokens, int64_t batch, int64_t max_q_len,
                                          int n_q_heads, int n_kv_heads, int head_dim) {
  if (max_q_len > tokens) max_q_len = tokens;
  // pieces are at most SMs where there are any, whatever the lengths
  const TcWork w = plan(tokens, batch, max_q_len, n_q_heads, n_kv_heads, int64_t(1) << 40);
  if (w.cells == 0) return 0;
  if (w.splits == 1) return 16;
  return static_cast<size_t>(w.cells) * w.splits * 2 * kRows *
         (static_cast<size_t>(head_dim) * 4 + 8);
}

cudaError_t launch_paged_attention_tc(const PagedAttnArgs& a, int dtype, void* workspace, bool pdl,
                                      cudaStream_t stream) {
  if (dtype == kDtypeBF16)
    return a.head_dim == 128 ? chunk_launch<__nv_bfloat16, 128>(a, workspace, pdl, stream)
                             : chunk_launch<__nv_bfloat16, 64>(a, workspace, pdl, stream);
  return a.head_dim == 128 ? chunk_launch<__half, 128>(a, workspace, pdl, stream)
                           : chunk_launch<__half, 64>(a, workspace, pdl, stream);
}

}  // namespace vl
