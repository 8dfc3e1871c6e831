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
//     has grown by more than 2^8 since the last time (2^4 in f16): until then
//     weights are taken about the old maximum, which fp32 sums and both 16-bit
//     types hold (see kLift).
//   * a warp each turns page ids into TMA boxes of K and of V, one thread
//     issues the MMAs, four warps scale and store finished rows while the
//     others are at the next cell, one warp walks along the cells.
// Cells (256 rows x kv head) lie on one line that the CTAs share equally.  A
// long cell is cut where a share ends, and a second launch joins the partial
// sums of its pieces.
//
// 2048 tokens after 14336, 16 / 4 heads of 128, bf16: 226 us at 1.9 GHz, 1140
// TFLOP/s, 0.69 of cuBLAS's burst rate; 265 where long runs settle under the
// power cap, 0.70 of its sustained rate.  What bounds it is the chain of a
// block's tile (maximum, exponentials, two products: some 4000 cycles for two
// blocks side by side, 2050 of them tensor cores' and 1940 the exponentials').
// Short cells add what they cost by themselves (16 x 383 tokens, 33.4 us: 9000
// cycles until the first scores, 3000 for a cell's last product and its rows,
// runs of 2 or 3 cells).
#include <cuda.h>

#include <atomic>
#include <cmath>

#include "vl_common.cuh"
#include "vl_kernels.h"
#include "vl_paged.cuh"
#include "vl_tma.cuh"

namespace vl {
namespace {

constexpr int kRows = 128;                // rows of a block (MMA M)
constexpr int kTile = 128;                // positions of a tile
constexpr int kStages = 2;                // of K and of V
constexpr int kSoftThreads = 256;         // two blocks' warps
constexpr int kEndWarp = 8;               // four warps that finish rows
constexpr int kQKWarp = 12;
constexpr int kMmaWarp = 13;
constexpr int kPlanWarp = 14;
constexpr int kVWarp = 15;
constexpr int kThreads = 512;
constexpr int kPlans = 4;                 // pieces that the walk is ahead
// How far a row's maximum may grow before O is rescaled, and what weights are
// held times of (log2): with both they reach 2^15 of the 65504 that f16 takes.
// So small ones keep their bits there down to 2^-25 of the largest and some
// down to 2^-35, where sums of thousands of them count beside one large
// weight.  Growth of 2^4 costs nothing against 2^8 (f16, 2048 tokens after 14336:
// 231.8 and 232.4 us), 2^2 some (236.8).  bf16 has fp32's exponents.
template <typename T>
constexpr float kRescaleLog2 = std::is_same<T, __half>::value ? 4.0f : 8.0f;
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 11.0f : 0.0f;

template <int HD>
struct Shape {
  static constexpr int kHalves = HD / 64;
  static constexpr int kColumn = kRows * 128;          // bytes: 128 rows x 64 dims
  static constexpr int kMatrix = kHalves * kColumn;    // 128 rows x HD
  static constexpr int kQ = 0;                         // two blocks
  static constexpr int kK = 2 * kMatrix;
  static constexpr int kV = kK + kStages * kMatrix;
  static constexpr int kOut = kV + kStages * kMatrix;  // 32 rows x 64 dims a finishing warp
  static constexpr int kSums = kOut + 4 * 4096;        // (max, sum) of two blocks' rows
  static constexpr int kBars = kSums + 2 * kRows * 8;
  static constexpr int kBytes = kBars + 1024 + 1024;    // barriers, and the ring's alignment
};

// A piece of work as the walk hands it to the others.
struct Plan {
  int row0;           // packed row of its first token
  int tokens;         // tokens from there to the sequence's end
  int seen0;          // positions that the first token sees, less one
  int len;            // positions of the sequence
  int h, b;           // kv head, sequence
  int j0, j1;         // tiles of positions
  int count[2];       // tiles of each block
  int whole;          // all tiles of its cell
  int last;           // no piece: the run is over
  int apart;          // the run is worth setting its two blocks apart
};

struct Bars {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t v_tail[kStages];
  uint64_t s_full[2], p_half[2], p_ready[2], o_done[2], o_free[2], sums_full[2],
      sums_free[2];
  uint64_t plan_full[kPlans], plan_empty[kPlans];
  uint64_t end;
  Plan plan[kPlans];
  uint32_t tmem;
  int bad;
};
static_assert(sizeof(Bars) <= 1024, "barrier block");

struct TcWork {
  float* part;        // [2 * grid][256 rows][HD]: a CTA's cut pieces
  float2* ml;         // [2 * grid][256] their (max, sum)
  int* next;          // [2 * grid] the slot that holds the cell's next piece, or -1
  struct CutCell* first;   // [grid] the cut cell that begins in a CTA
};

struct CutCell {
  int row0, tokens, h;   // as in Plan
  int cut;               // 0: none
};

// A cell is a pair of blocks of one sequence and kv head against the n tiles
// of positions that they see.  All cells lie on one line, by sequence and head
// (a head's pairs in the order of cells_before), each as long as the positions it sees plus what a cell
// costs by itself, so that places are sums in closed form; CTAs take equal
// runs of the line.  Where a run ends inside a cell the cell is cut, at a
// whole tile, if both ends are worth a piece; else it goes to the side that
// has more of it.
constexpr int kCellCost = 2 * kTile;      // of a cell by itself, in positions
// A run of this many positions sets its blocks half a tile apart, which costs
// it 1.5 us at the start: 16 x 383 tokens (1245 a run) 34.1 us set apart, 33.3
// in step; 23 ragged sequences (4000) 88 and 95 us.
constexpr int64_t kApart = 16 * kTile;
// Shortest piece of a cut cell.  23 ragged sequences: 93.5 us with three tiles,
// 95.4 with four, 93.9 with two (and 104 with cells that cost 192 positions).
constexpr int kMinPiece = 3;              // tiles

// Where a walk along the line stands.
struct Walk {
  int b;              // sequence (batch: past the end)
  SeqView s;
  int past;           // positions before the new tokens
  int h, u;           // kv head, place in its order of pairs of blocks
  int t;              // that pair
  int pairs;          // of the sequence
  int64_t at, size;   // the cell's place on the line
  int n;              // its tiles
  int rows_tok;       // tokens of a block
  int j0, j1;         // this CTA's tiles of it
};

__device__ __forceinline__ int cut_at(int64_t x, const Walk& w) {
  const int64_t into = x - w.at;
  if (into <= 0) return 0;
  if (into >= w.size) return w.n;
  if (w.n < 2 * kMinPiece) return 2 * into >= w.size ? w.n : 0;
  const int j = into < kCellCost ? 0 : static_cast<int>((into - kCellCost) / kTile);
  return j < kMinPiece ? 0 : (w.n - j < kMinPiece ? w.n : j);
}

__device__ __forceinline__ int tiles_seen(const SeqView& s, int last_token) {
  const int see = s.len - s.rows + last_token;         // positions of that token
  return s.len > 0 && see > 0 ? (see + kTile - 1) / kTile : 0;
}
// A head's first u cells on the line.  Its pairs come as last, first, last but
// one, second, ...: two neighbours add up to the same, so that runs of few
// whole cells differ less (16 x 383 tokens: 35.7 -> 34.5 us).
__device__ __forceinline__ int64_t cells_before(int past, int rows, int pairs, int u, int pair) {
  const int64_t each = static_cast<int64_t>(past) + kCellCost, c = u >> 1;
  int64_t size = u * each + (c * (pairs + 1) + ((u & 1) ? pairs - c : 0)) * pair;
  if (u > 0) size -= pairs * static_cast<int64_t>(pair) - rows;   // the last is shorter
  return size;
}
__device__ __forceinline__ int64_t head_size(const SeqView& s, int pair) {
  if (s.rows == 0) return 0;
  const int past = max(0, s.len - s.rows), pairs = (s.rows + pair - 1) / pair;
  return cells_before(past, s.rows, pairs, pairs, pair);
}

// The line's length; before: where the sequences that this lane adds up
// begin (a whole warp, the l-th 32nd of them each).
__device__ __forceinline__ int64_t line_length(const PagedAttnArgs& a, int shift, int pair,
                                               int lane, int64_t* before, bool* bad) {
  const int each = (a.batch + 31) / 32;
  const int b0 = min(a.batch, lane * each), b1 = min(a.batch, b0 + each);
  int64_t mine = 0;
  *bad = false;
  for (int b = b0; b < b1; ++b) {
    const SeqView s = sequence_view(a, b, shift);
    *bad |= s.bad;
    mine += head_size(s, pair) * a.n_kv_heads;
  }
  int64_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t n = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += n;
  }
  *before = upto - mine;
  return __shfl_sync(0xffffffffu, upto, 31);
}

__device__ __forceinline__ void enter_cell(int pair, Walk& w) {
  w.t = (w.u & 1) ? w.u >> 1 : w.pairs - 1 - (w.u >> 1);
  const int last = min(w.s.rows, (w.t + 1) * pair);
  w.n = tiles_seen(w.s, last);
  w.size = static_cast<int64_t>(w.past) + last + kCellCost;
}
// The next sequence from w.b on that has rows.
__device__ __forceinline__ void enter_sequence(const PagedAttnArgs& a, int shift, int pair,
                                               Walk& w) {
  for (; w.b < a.batch; ++w.b) {
    w.s = sequence_view(a, w.b, shift);
    if (w.s.rows > 0) break;
  }
  w.h = w.u = 0;
  if (w.b == a.batch) return;
  w.past = max(0, w.s.len - w.s.rows);
  w.pairs = (w.s.rows + pair - 1) / pair;
  enter_cell(pair, w);
}
__device__ __forceinline__ void next_cell(const PagedAttnArgs& a, int shift, int pair, Walk& w) {
  w.at += w.size;
  if (++w.u == w.pairs) {
    w.u = 0;
    if (++w.h == a.n_kv_heads) {
      ++w.b;
      enter_sequence(a, shift, pair, w);
      return;
    }
  }
  enter_cell(pair, w);
}
// The cell that holds place x.
__device__ __forceinline__ Walk find_cell(const PagedAttnArgs& a, int shift, int pair,
                                          int64_t before, int64_t x) {
  const int owner = 31 - __clz(__ballot_sync(0xffffffffu, before <= x));
  Walk w;
  w.b = owner * ((a.batch + 31) / 32);
  w.at = __shfl_sync(0xffffffffu, before, owner);
  w.rows_tok = pair / 2;
  enter_sequence(a, shift, pair, w);
  while (w.b < a.batch) {
    const int64_t head = head_size(w.s, pair), into = x - w.at;
    if (into < head * a.n_kv_heads) {
      w.h = static_cast<int>(divide(into, head));
      w.at += w.h * head;
      int hi = w.pairs;                   // the last cell of the head that begins at or before x
      while (hi - w.u > 1) {
        const int mid = (w.u + hi) / 2;
        if (w.at + cells_before(w.past, w.s.rows, w.pairs, mid, pair) <= x) w.u = mid;
        else hi = mid;
      }
      w.at += cells_before(w.past, w.s.rows, w.pairs, w.u, pair);
      enter_cell(pair, w);
      break;
    }
    w.at += head * a.n_kv_heads;
    ++w.b;
    enter_sequence(a, shift, pair, w);
  }
  return w;
}

// This CTA's run, cell by cell.
struct Run {
  int64_t x0, x1;
  int shift, pair;
};
__device__ __forceinline__ bool settle(const PagedAttnArgs& a, const Run& r, Walk& w) {
  for (; w.b < a.batch && w.at < r.x1; next_cell(a, r.shift, r.pair, w)) {
    w.j0 = cut_at(r.x0, w);
    w.j1 = cut_at(r.x1, w);
    if (w.j1 > w.j0) return true;
    if (w.n == 0 && w.at >= r.x0) return true;
  }
  return false;
}
// Tiles of block i within the piece.
__device__ __forceinline__ int block_tiles(const Walk& w, int i) {
  const int first = w.t * 2 * w.rows_tok + i * w.rows_tok;
  if (first >= w.s.rows) return 0;
  return max(0, min(w.j1, tiles_seen(w.s, min(w.s.rows, first + w.rows_tok))) - w.j0);
}

// The slow side of a wait: bounded, and given up when another has run out.
__device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity, int* bad) {
  for (uint32_t i = 0; i < kWaitPolls; ++i) {
    if (mbarrier_test(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(bad)) return false;
  }
  atomicExch(bad, 1);
  return false;
}
__device__ __forceinline__ bool wait_or_bad(uint64_t* bar, uint32_t parity, int* bad) {
  const uint32_t at = smem_addr(bar);
  return mbarrier_test(at, parity) || wait_longer(at, parity, bad);
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
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
__device__ __forceinline__ float max3(uint32_t a, uint32_t b, uint32_t c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;"
      : "=f"(y)
      : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)), "f"(__uint_as_float(c)));
  return y;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// 2^x of two values on the multiply-add pipe, beside the exponential unit:
// x = n + f with |f| <= 1/2, a degree-5 polynomial of f (least squares of the
// relative error, reweighted until it is level: 2.2e-7 in fp32), n added to the
// exponent.  Values below -126 give
// about 1e-38 (a row all of -inf is told by its maximum), NaN gives what rounds
// to infinity in either type.
__device__ __forceinline__ float2 ex2_pair(float2 z) {
  const uint64_t t = pair_of(max_or_nan(z.x, -126.0f), max_or_nan(z.y, -126.0f));
  constexpr float kRound = 12582912.0f;   // 1.5 * 2^23: the sum's low bits are n
  const uint64_t r = add2(t, pair_of(kRound, kRound));
  const uint64_t f = fma2(add2(r, pair_of(-kRound, -kRound)), pair_of(-1.0f, -1.0f), t);
  uint64_t p = fma2(pair_of(0.0013276471f, 0.0013276471f), f, pair_of(0.009675541f, 0.009675541f));
  p = fma2(p, f, pair_of(0.05550713f, 0.05550713f));
  p = fma2(p, f, pair_of(0.2402212f, 0.2402212f));
  p = fma2(p, f, pair_of(0.69314694f, 0.69314694f));
  p = fma2(p, f, pair_of(1.0000001f, 1.0000001f));
  const float2 pf = halves_of(p), rf = halves_of(r);
  return make_float2(__uint_as_float(__float_as_uint(pf.x) + (__float_as_uint(rf.x) << 23)),
                     __uint_as_float(__float_as_uint(pf.y) + (__float_as_uint(rf.y) << 23)));
}
// Which of the 32 pairs of half a row go that way: one in four.  A row's 128
// exponentials then take 1190 cycles with one warp on a scheduler and 1940
// with two, against 1360 and 2240 with none, 1350 and 2040 with three of
// eight.
__device__ constexpr bool by_polynomial(int pair) { return pair % 4 == 1; }

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
  float2* sums = reinterpret_cast<float2*>(smem_raw + (base - raw0) + L::kSums);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int shift = ilog2(a.page_size);
  const int G = a.n_q_heads / a.n_kv_heads;

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbarrier_init(&bars.k_full[s], 1);
      mbarrier_init(&bars.k_empty[s], 1);
      mbarrier_init(&bars.v_full[s], 1);
      mbarrier_init(&bars.v_empty[s], 1);
      mbarrier_init(&bars.v_tail[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbarrier_init(&bars.q_full[i], 1);
      mbarrier_init(&bars.q_empty[i], 1);
      mbarrier_init(&bars.s_full[i], 1);
      mbarrier_init(&bars.p_half[i], kSoftThreads / 64);    // a block's warps
      mbarrier_init(&bars.p_ready[i], kSoftThreads / 64);
      mbarrier_init(&bars.o_done[i], 1);
      mbarrier_init(&bars.o_free[i], 4);                    // the finishing warps
      mbarrier_init(&bars.sums_full[i], kSoftThreads / 64);
      mbarrier_init(&bars.sums_free[i], 4);
    }
    for (int k = 0; k < kPlans; ++k) {
      mbarrier_init(&bars.plan_full[k], 1);
      mbarrier_init(&bars.plan_empty[k], 3 + kSoftThreads / 32 + 4);   // every reader's warp
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
  if (warp == kQKWarp && elect_lane()) {
    prefetch_map(&qmap);
    prefetch_map(&kmap);
    prefetch_map(&vmap);
  }
  __syncwarp();
  // The planning warp looks the lengths up while the others set up; they and
  // the tables are not written by the kernel before this one.
  Run run;
  Walk at;
  int64_t share = 0;
  if (warp == kPlanWarp) {
    run.shift = shift;
    run.pair = 2 * (kRows / G);
    int64_t before;
    bool bad_lengths;
    const int64_t total = line_length(a, shift, run.pair, lane, &before, &bad_lengths);
    if (bad_lengths && blockIdx.x == 0 && a.status) atomicOr(a.status, VL_STATUS_BAD_PAGE);
    share = divide(total + gridDim.x - 1, gridDim.x);
    run.x0 = min(total, blockIdx.x * share);
    run.x1 = min(total, run.x0 + share);
    at.b = a.batch;
    if (run.x0 < run.x1) at = find_cell(a, shift, run.pair, before, run.x0);
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = bars.tmem;

  // Pieces as they come, for the producer, the MMA warp and the softmax warps.
  uint32_t piece = 0;
  bool ok = true;
  auto take = [&](Plan& p) {
    ok = wait_or_bad(&bars.plan_full[piece % kPlans], (piece / kPlans) & 1, &bars.bad);
    if (!ok) return false;
    p = bars.plan[piece % kPlans];
    __syncwarp();
    if (lane == 0) mbarrier_arrive(&bars.plan_empty[piece % kPlans]);
    ++piece;
    return p.last == 0;
  };

  if (warp == kPlanWarp) {
    // ---- the walk ----
    CutCell begins{};
    pdl_wait();                                        // the join before may be reading
    for (bool more = true; more; ++piece) {
      more = settle(a, run, at);
      const int slot = piece % kPlans;
      if (piece >= kPlans &&
          !wait_or_bad(&bars.plan_empty[slot], ((piece / kPlans) & 1) ^ 1, &bars.bad))
        break;
      if (lane == 0) {
        Plan p{};
        p.last = !more;
        if (more) {
          const int tok0 = 2 * at.t * at.rows_tok;
          p.row0 = at.s.start + tok0;
          p.tokens = at.s.rows - tok0;
          p.seen0 = at.s.len - at.s.rows + tok0;
          p.len = at.s.len;
          p.h = at.h;
          p.b = at.b;
          p.j0 = at.j0;
          p.j1 = at.j1;
          p.count[0] = block_tiles(at, 0);
          p.count[1] = block_tiles(at, 1);
          p.apart = share >= kApart;
          p.whole = at.j0 == 0 && at.j1 == at.n;
          if (!p.whole) {
            // a CTA's first piece may begin inside its cell (slot 0), its last end there
            int then = -1;
            if (at.j1 < at.n) {
              int cta = blockIdx.x + 1;
              while (cut_at((cta + 1) * share, at) == at.j1) ++cta;
              then = 2 * cta;
            }
            w.next[2 * blockIdx.x + (at.j0 > 0 ? 0 : 1)] = then;
            if (at.j0 == 0) begins = CutCell{p.row0, p.tokens, p.h, 1};
          }
        }
        bars.plan[slot] = p;
        mbarrier_arrive(&bars.plan_full[slot]);
      }
      __syncwarp();
      if (more) next_cell(a, shift, run.pair, at);
    }
    if (lane == 0) w.first[blockIdx.x] = begins;
    // the last ones have been read before this block goes
    for (uint32_t k = piece < kPlans ? 0 : piece - kPlans; k < piece; ++k)
      if (!wait_or_bad(&bars.plan_empty[k % kPlans], (k / kPlans) & 1, &bars.bad)) break;
  } else if (warp == kQKWarp || warp == kVWarp) {
    // ---- copies: one warp Q of a piece and its K tiles, another the V tiles ----
    const bool qk = warp == kQKWarp;
    pdl_wait();
    if (qk) pdl_release();
    const int box_rows = 1 << box_shift, rows_tok = kRows / G;
    const int boxes = kTile >> box_shift;              // of a tile: 1 .. 8
    uint64_t* const full = qk ? bars.k_full : bars.v_full;
    uint64_t* const empty = qk ? bars.k_empty : bars.v_empty;
    const CUtensorMap* const map = qk ? &kmap : &vmap;
    const uint32_t ring = base + (qk ? L::kK : L::kV);
    uint32_t tile = 0, asked[2] = {0, 0};              // tiles and Q blocks so far
    // Rows of V past a sequence's end hold anything: their weights are 0, and
    // so must they be.  The tile is cleared there once it has arrived, while
    // the next one is on its way, and only then handed on.
    uint32_t tails = 0;                                // a bit a stage: its next parity
    int clear = kTile, clear_stage = 0;                // the first row to clear
    auto clear_tail = [&] {
      if (clear == kTile) return;
      ok = wait_or_bad(&bars.v_tail[clear_stage], (tails >> clear_stage) & 1, &bars.bad);
      tails ^= 1u << clear_stage;
      const uint32_t v = ring + clear_stage * L::kMatrix;
      for (int z = lane; z < (kTile - clear) * (HD / 8); z += 32) {
        const int row = clear + z / (HD / 8), ch = z % (HD / 8);
        asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(
                         v + (ch >> 3) * L::kColumn + row * 128 + (((ch & 7) ^ (row & 7)) << 4)),
                     "r"(0)
                     : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&full[clear_stage]);
      clear = kTile;
    };
    Plan p;
    while (ok && take(p)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!qk || !ok || p.count[i] == 0) continue;
        if (asked[i] > 0) ok = wait_or_bad(&bars.q_empty[i], (asked[i] - 1) & 1, &bars.bad);
        if (!ok) continue;
        ++asked[i];
        if (elect_lane()) {
          mbarrier_expect(&bars.q_full[i], L::kHalves * 128 * G * rows_tok);
#pragma unroll
          for (int c = 0; c < L::kHalves; ++c)
            tma_load_3d(base + L::kQ + i * L::kMatrix + c * L::kColumn, &qmap, c * 64, p.h * G,
                        p.row0 + i * rows_tok, &bars.q_full[i]);
        }
        __syncwarp();
      }
      int page = 0, at_box = 32;                       // pages of 32 boxes, and the tile's first
      for (int j = p.j0; ok && j < p.j1; ++j, ++tile, at_box += boxes) {
        const int pos0 = j * kTile;
        if (at_box == 32) {
          at_box = 0;
          // (a box that far ahead may begin past 2^31: only its distance is formed)
          const int ahead = lane << box_shift;
          if (ahead < min(p.len, p.j1 * kTile) - pos0) {
            page = a.page_table[p.b * a.table_stride + ((pos0 + ahead) >> shift)];
            if (page < 0 || page >= a.num_pages) {     // read as rows of zeros
              page = static_cast<int>(a.num_pages);
              if (a.status) atomicOr(a.status, VL_STATUS_BAD_PAGE);
            }
          }
        }
        const int need = (min(kTile, p.len - pos0) + box_rows - 1) >> box_shift;
        const int st = tile % kStages;
        if (tile >= kStages) ok = wait_or_bad(&empty[st], ((tile / kStages) & 1) ^ 1, &bars.bad);
        if (!ok) break;
        int pk[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) pk[k] = __shfl_sync(0xffffffffu, page, (at_box + k) & 31);
        const bool tail = !qk && p.len - pos0 < kTile;
        uint64_t* const landed = tail ? &bars.v_tail[st] : &full[st];
        if (elect_lane()) {
          mbarrier_expect(landed, static_cast<uint32_t>(need) * box_rows * 128 * L::kHalves);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (k >= need) break;
            const uint32_t dst = ring + st * L::kMatrix + k * box_rows * 128;
            const int row = (pos0 + (k << box_shift)) & (a.page_size - 1);
#pragma unroll
            for (int c = 0; c < L::kHalves; ++c)
              tma_load_4d(dst + c * L::kColumn, map, c * 64, p.h, row, pk[k], landed);
          }
        }
        __syncwarp();
        clear_tail();
        if (tail) {
          clear = p.len - pos0;
          clear_stage = st;
        }
      }
      // a piece without tiles: the plan behind it may wait for the last one's rows
      if (ok && p.j0 == p.j1) clear_tail();
    }
    if (ok) clear_tail();
    if (*reinterpret_cast<volatile int*>(&bars.bad)) {
      // leave no copy in flight (each wait is bounded; what was never asked
      // for lets it run out)
      auto drain = [&](uint64_t* bar, uint32_t parity) {
        for (int i = 0; i < 1000 && !mbarrier_test(bar, parity); ++i) {}
      };
      for (int i = 0; i < 2; ++i)
        if (asked[i] > 0) drain(&bars.q_full[i], (asked[i] - 1) & 1);
      for (uint32_t t = tile < kStages ? 0 : tile - kStages; t <= tile; ++t)
        drain(&full[t % kStages], (t / kStages) & 1);
      if (clear < kTile) drain(&bars.v_tail[clear_stage], (tails >> clear_stage) & 1);
    }
  } else if (warp == kMmaWarp) {
    // ---- products: one thread ----
    // Each block is a stream of tiles of its own, across cells: S of its next
    // tile is issued behind P V of the last, whatever the other block does.
    // This thread's own steps are on every tile's critical path, so
    // descriptors are made once and only their low words move.
    if (elect_lane()) {
      constexpr uint32_t kIdescS = instruction<T>(kTile, false);
      constexpr uint32_t kIdescO = instruction<T>(HD, true);
      uint64_t qd[2], kd[kStages], vd[kStages];
#pragma unroll
      for (int i = 0; i < 2; ++i) qd[i] = desc(base + L::kQ + i * L::kMatrix, 16, 1024);
#pragma unroll
      for (int i = 0; i < kStages; ++i) {
        kd[i] = desc(base + L::kK + i * L::kMatrix, 16, 1024);
        vd[i] = desc(base + L::kV + i * L::kMatrix, L::kColumn, 1024);
      }
      uint32_t tile = 0, heads[2] = {0, 0}, used[2] = {0, 0}, begun[2] = {0, 0};
      auto wait = [&](uint64_t& bar, uint32_t parity) {
        ok = ok && wait_or_bad(&bar, parity & 1, &bars.bad);
      };
      auto ask = [&](int i, uint32_t t, bool first, bool last) {   // S_i = Q_i K^T of tile t
        if (first) wait(bars.q_full[i], heads[i]++);
        wait(bars.k_full[t % kStages], t / kStages);
        if (!ok) return;
        fence_after();
        const uint64_t k = kd[t % kStages];
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = ((kk >> 2) * L::kColumn + (kk & 3) * 32) >> 4;
          mma_ss(tmem + i * kTile, qd[i] + off, k + off, kIdescS, kk > 0);
        }
        commit(&bars.s_full[i]);
        if (last) commit(&bars.q_empty[i]);
      };
      // O_i (+)= P_i V over one half of the tile's positions
      auto values = [&](int i, int half, bool first) {
        const uint64_t v = vd[tile % kStages] + half * (kTile / 2 * 128 >> 4);
        const uint32_t p = tmem + i * kTile + half * (kTile / 4);
        fence_after();
#pragma unroll
        for (int kk = 0; kk < kTile / 32; ++kk)
          mma_ts(tmem + 2 * kTile + i * HD, p + kk * 8, v + kk * (2048 >> 4), kIdescO,
                 !first || kk > 0);
      };
      // tiles of a piece, and of its blocks (a piece without tiles is not ours)
      struct Count {
        int all, of[2], apart;
      };
      auto next_piece = [&](Count& c) {                    // false: the run is over
        wait(bars.plan_full[piece % kPlans], piece / kPlans);
        if (!ok) return false;
        const Plan& p = bars.plan[piece % kPlans];
        const bool over = p.last != 0;
        c.all = p.j1 - p.j0;
        c.apart = p.apart;
        c.of[0] = p.count[0];
        c.of[1] = p.count[1];
        mbarrier_arrive(&bars.plan_empty[piece % kPlans]);
        ++piece;
        return !over;
      };
      Count now, then;
      bool more = true;
      while (ok && more) {                // pieces with tiles, one behind the other
        more = next_piece(now);
        if (!more || now.all == 0) continue;
        if (now.of[0] > 0) {
          ask(0, tile, true, now.of[0] == 1);
          // in a long run the second block starts half a tile later, and stays
          // there: one's products run under the other's exponentials
          if (tile == 0 && now.apart) wait(bars.p_half[0], 0);
        }
        if (now.of[1] > 0) ask(1, tile, true, now.of[1] == 1);
        commit(&bars.k_empty[tile % kStages]);
        int jj = 0;
        bool linked = true;               // the next tile's scores are asked for
        while (ok && linked) {
          const bool ends = jj + 1 == now.all;
          int jn = jj + 1;
          then = now;
          if (ends) {
            // One piece is looked ahead.  Where its rows see nothing, one with
            // tiles is looked for when this one's products are issued: plans are
            // handed out as far as kPlans ahead of the rows being finished.
            more = next_piece(then);
            linked = more && then.all > 0;
            jn = 0;
            if (!linked) then.of[0] = then.of[1] = 0;
          }
          wait(bars.v_full[tile % kStages], tile / kStages);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (jj < now.of[i]) {
              // O of the block's last cell has been read
              if (jj == 0 && begun[i]++ > 0) wait(bars.o_free[i], begun[i]);
              wait(bars.p_half[i], used[i]);
              if (ok) values(i, 0, jj == 0);
              wait(bars.p_ready[i], used[i]++);
              if (ok) {
                values(i, 1, false);
                if (jj + 1 == now.of[i]) commit(&bars.o_done[i]);
              }
            }
            if (jn < then.of[i]) ask(i, tile + 1, ends, jn + 1 == then.of[i]);
          }
          commit(&bars.v_empty[tile % kStages]);
          if (linked) commit(&bars.k_empty[(tile + 1) % kStages]);
          ++tile;
          now = then;
          jj = jn;
        }
      }
      // every MMA has ended, and with it the arrivals that it owes
      commit(&bars.end);
      (void)mbarrier_wait(&bars.end, 0);
    }
    __syncwarp();
  } else if (warp >= kEndWarp && warp < kEndWarp + 4) {
    // ---- rows of a piece, while the softmax warps are at the next one ----
    pdl_wait();                                        // it writes rows
    const int r = tid - kEndWarp * 32;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int rows_tok = kRows / G, g = r % G;
    const uint32_t stage = base + L::kOut + (warp - kEndWarp) * 4096;
    uint32_t finished[2] = {0, 0};
    Plan p;
    while (ok && take(p)) {
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const int count = i ? p.count[1] : p.count[0], tok = i * rows_tok + r / G;
        const bool mine = r < G * rows_tok && tok < p.tokens;
        if (!(ok = wait_or_bad(&bars.sums_full[i], (piece - 1) & 1, &bars.bad))) break;
        const float2 ml = sums[i * kRows + r];
        __syncwarp();
        if (lane == 0) mbarrier_arrive(&bars.sums_free[i]);
        float inv = 0.0f;
        if (count > 0) {
          uint32_t& n = i ? finished[1] : finished[0];
          if (!(ok = wait_or_bad(&bars.o_done[i], n & 1, &bars.bad))) break;
          ++n;
          fence_after();
          // (a sum that is NaN stays so; a row all of -inf is a row of zeros)
          inv = ml.y != ml.y || ml.x > -INFINITY ? 1.0f / ml.y : 0.0f;
        }
        const int64_t row256 =
            (2 * static_cast<int64_t>(blockIdx.x) + (p.j0 > 0 ? 0 : 1)) * 2 * kRows + i * kRows + r;
        if (!p.whole && mine) w.ml[row256] = ml;
        const int64_t at_row = static_cast<int64_t>(p.row0 + tok) * a.out_row_stride +
                               static_cast<int64_t>(p.h * G + g) * HD;
        const uint32_t to = tmem + 2 * kTile + i * HD + lanes;
#pragma unroll 1
        for (int c = 0; c < HD; c += 64) {
          uint32_t o[64];
          if (count > 0) {
            tmem_load32(to + c, o);
            tmem_load32(to + c + 32, o + 32);
            tmem_load_wait<64>(o);
            if (c + 64 == HD) {
              fence_before();
              __syncwarp();
              if (lane == 0) mbarrier_arrive(&bars.o_free[i]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 64; ++e) o[e] = 0;
          }
          if (!p.whole) {
            if (mine) {
              float4* dst = reinterpret_cast<float4*>(w.part + row256 * HD + c);
#pragma unroll
              for (int e = 0; e < 16; ++e)
                dst[e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                     __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
            }
            continue;
          }
          // A lane has a row; a store of 32 rows at once would touch 32
          // half-filled sectors.  Through shared memory eight lanes take a
          // row's 128 bytes instead.
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(o[8 * v + e]) * inv;
            const uint4 y = S::pack(f);
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(
                             stage + lane * 128 + ((v ^ (lane & 7)) << 4)),
                         "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w)
                         : "memory");
          }
          __syncwarp();
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            const int row = v * 4 + (lane >> 3), ch = lane & 7;
            uint4 y;
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                         : "r"(stage + row * 128 + ((ch ^ (row & 7)) << 4))
                         : "memory");
            const int64_t to_row = __shfl_sync(0xffffffffu, mine ? at_row : -1, row);
            if (to_row >= 0) st_vec(static_cast<T*>(a.out) + to_row + c + ch * 8, y);
          }
          __syncwarp();
        }
      }
    }
    if (!ok && r == 0 && a.status) atomicOr(a.status, VL_STATUS_TIMEOUT);
  } else {
    // ---- softmax: a thread per row ----
    const int i = warp >> 2;                           // block
    const int r = tid & (kRows - 1);
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + i * kTile + lanes, to = tmem + 2 * kTile + i * HD + lanes;
    const float scale = a.scale * kLog2e;
    const int rows_tok = kRows / G, tok = i * rows_tok + r / G;
    uint32_t used = 0;
    Plan p;
    while (ok && take(p)) {
      const int count = i ? p.count[1] : p.count[0];
      const bool mine = r < G * rows_tok && tok < p.tokens;
      // (rows of nobody are not hidden: their results go nowhere)
      const int see = !mine ? 0x7fffffff : (p.len > 0 ? p.seen0 + tok + 1 : 0);
      float m = -INFINITY, l = 0.0f;
      for (int jj = 0; jj < count; ++jj) {
        if (!(ok = wait_or_bad(&bars.s_full[i], used & 1, &bars.bad))) break;
        ++used;
        fence_after();
        const int pos0 = (p.j0 + jj) * kTile;
        // Half a row at a time, read from tensor memory once for the maximum
        // and again for the weights: a load takes some 40 cycles, and held
        // rows (128 registers) and unrolled code (instruction fetches, which
        // short chunks do not amortise) cost more.
        const bool cut = __any_sync(0xffffffffu, pos0 + kTile > see);
        float mx = -INFINITY, my = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < kTile; c += kTile / 2) {
          uint32_t x[kTile / 2];
          tmem_load32(ts + c, x);
          tmem_load32(ts + c + 32, x + 32);
          tmem_load_wait<kTile / 2>(x);
          if (cut) {
            hide<kTile / 2>(x, see - pos0 - c);
            tmem_store32(ts + c, x);      // for the second reading
            tmem_store32(ts + c + 32, x + 32);
            tmem_store_wait();
          }
          float mz = max3(x[0], x[1], x[2]), mw = max3(x[3], x[4], x[5]);
#pragma unroll
          for (int e = 6; e + 8 <= kTile / 2; e += 8) {
            mx = max3(__float_as_uint(mx), x[e], x[e + 1]);
            my = max3(__float_as_uint(my), x[e + 2], x[e + 3]);
            mz = max3(__float_as_uint(mz), x[e + 4], x[e + 5]);
            mw = max3(__float_as_uint(mw), x[e + 6], x[e + 7]);
          }
          mx = max3(__float_as_uint(mx), x[kTile / 2 - 2], x[kTile / 2 - 1]);
          my = fmaxf(my, fmaxf(mz, mw));
        }
        mx = fmaxf(mx, my);
        // Rounded so that no weight passes 2^(kLift + kRescaleLog2), however large
        // the scores (past 2^24 a rounding is more than 1).
        mx = __fmul_ru(mx, scale);
        if (__any_sync(0xffffffffu, mine && mx > __fadd_rd(m, kRescaleLog2<T>))) {
          const float m_new = fmaxf(m, mx);
          const float f = m_new == -INFINITY ? 1.0f : ex2(m - m_new);
          l *= f;
          m = m_new;
          if (jj > 0) {
            // the products that wrote O are done: this tile's scores were
            // issued behind them
#pragma unroll 1
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
        const float off = m == -INFINITY ? 0.0f : __fsub_rd(kLift<T>, m);
        const uint64_t scale2 = pair_of(scale, scale), off2 = pair_of(off, off);
        // P rounds to the storage type, as its tensor-core operand: half a
        // step per weight, against a sum that stays in fp32
        uint64_t sum[2] = {0, 0};
#pragma unroll 1
        for (int c = 0; c < kTile; c += kTile / 2) {
          uint32_t x[kTile / 2], pk[kTile / 4];
          tmem_load32(ts + c, x);
          tmem_load32(ts + c + 32, x + 32);
          tmem_load_wait<kTile / 2>(x);
          if (cut) {                      // weights that are exactly 0
#pragma unroll
            for (int e = 0; e < kTile / 2; e += 2) {
              const float2 z = halves_of(fma2(pair_of(x[e], x[e + 1]), scale2, off2));
              const float e0 = ex2(z.x), e1 = ex2(z.y);
              sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pair_of(e0, e1));
              pk[e / 2] = pack16(e0, e1, T());
            }
          } else {
#pragma unroll
            for (int e = 0; e < kTile / 2; e += 2) {
              const uint64_t z2 = fma2(pair_of(x[e], x[e + 1]), scale2, off2);
              const float2 z = halves_of(z2);
              float e0, e1;
              if (by_polynomial(e / 2)) {
                const float2 y = ex2_pair(z);
                e0 = y.x;
                e1 = y.y;
              } else {
                e0 = ex2(z.x);
                e1 = ex2(z.y);
              }
              sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], pair_of(e0, e1));
              pk[e / 2] = pack16(e0, e1, T());
            }
          }
          tmem_store32(ts + c / 2, pk);   // over columns that have been read
          // the products over these positions may start
          tmem_store_wait();
          fence_before();
          __syncwarp();
          if (lane == 0) mbarrier_arrive(c == 0 ? &bars.p_half[i] : &bars.p_ready[i]);
        }
        const float2 s0 = halves_of(add2(sum[0], sum[1]));
        l += s0.x + s0.y;
      }
      if (!ok) break;
      // maximum and sum of the rows, for the warps that finish them
      if (piece > 1 && !(ok = wait_or_bad(&bars.sums_free[i], piece & 1, &bars.bad))) break;
      sums[i * kRows + r] = make_float2(m, l);
      __syncwarp();
      if (lane == 0) mbarrier_arrive(&bars.sums_full[i]);
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

// Joins the pieces of the cut cell that begins in CTA blockIdx.x, in order: a
// warp per row.
constexpr int kJoinBlocks = 8;
constexpr int kMaxPieces = 1024;          // of a cell: at most one per CTA
template <typename T, int HD>
__global__ void __launch_bounds__(256)
    paged_chunk_join_kernel(const __grid_constant__ PagedAttnArgs a, TcWork w) {
  using S = Storage<T>;
  constexpr int E = HD / 32;              // dims of a lane
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.n_q_heads / a.n_kv_heads, rows_tok = kRows / G;
  __shared__ int slots[kMaxPieces];
  __shared__ int pieces;
  pdl_wait();
  const CutCell c = w.first[blockIdx.x];
  if (c.cut == 0) return;
  if (threadIdx.x == 0) {
    int n = 0;
    for (int slot = 2 * blockIdx.x + 1; slot >= 0 && n < kMaxPieces; slot = __ldcg(w.next + slot))
      slots[n++] = slot;
    pieces = n;
  }
  __syncthreads();
  for (int rr = blockIdx.y * 8 + warp; rr < 2 * kRows; rr += kJoinBlocks * 8) {
    const int r = rr % kRows, tok = rr / kRows * rows_tok + r / G, g = r % G;
    if (r >= G * rows_tok || tok >= c.tokens) continue;
    float M = -INFINITY, sum = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    for (int k = 0; k < pieces; ++k) {
      const int64_t row = static_cast<int64_t>(slots[k]) * 2 * kRows + rr;
      const float2 ml = __ldcg(w.ml + row);
      float y[E];
      if (E == 4) {
        const float4 q = __ldcg(reinterpret_cast<const float4*>(w.part + row * HD) + lane);
        y[0] = q.x, y[1] = q.y, y[E - 2] = q.z, y[E - 1] = q.w;
      } else {
        const float2 q = __ldcg(reinterpret_cast<const float2*>(w.part + row * HD) + lane);
        y[0] = q.x, y[1] = q.y;
      }
      // The row sees nothing of it, or scores of -inf alone; a NaN beside those
      // leaves a sum of NaN or, by the polynomial, one of 3e38.
      if (ml.x == -INFINITY && ml.y < 1.0f) continue;
      const float m_new = fmaxf(M, ml.x);
      const float f0 = exp2f(M - m_new), f1 = exp2f(ml.x - m_new);
      M = m_new;
      sum = sum * f0 + ml.y * f1;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * f0 + y[e] * f1;
    }
    const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(c.row0 + tok) * a.out_row_stride +
             static_cast<int64_t>(c.h * G + g) * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = S::from_float(o[e] * inv);
  }
}

int chunk_grid() { return sm_count() < kMaxPieces ? sm_count() : kMaxPieces; }

template <typename T, int HD>
cudaError_t chunk_launch(const PagedAttnArgs& a, void* workspace, bool pdl, cudaStream_t stream) {
  const int G = a.n_q_heads / a.n_kv_heads;
  TcWork w;
  const int64_t rows = static_cast<int64_t>(chunk_grid()) * 2 * 2 * kRows;
  w.ml = static_cast<float2*>(workspace);
  w.part = reinterpret_cast<float*>(w.ml + rows);
  w.first = reinterpret_cast<CutCell*>(w.part + rows * HD);
  w.next = reinterpret_cast<int*>(w.first + chunk_grid());
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
  const int grid = chunk_grid();
  e = launch_kernel(kernel, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem, stream, pdl, a,
                    qmap, kmap, vmap, w, box_shift);
  // a table too short for a cell that could be cut needs no join
  if (e != cudaSuccess ||
      static_cast<int64_t>(a.max_pages) * a.page_size <= (2 * kMinPiece - 1) * kTile)
    return e;
  return launch_kernel(paged_chunk_join_kernel<T, HD>,
                       dim3(static_cast<unsigned>(grid), kJoinBlocks), dim3(256), 0, stream, true,
                       a, w);
}

}  // namespace

size_t paged_attention_tc_workspace_bytes(int head_dim) {
  return static_cast<size_t>(chunk_grid()) * 2 * 2 * kRows *
             (static_cast<size_t>(head_dim) * 4 + sizeof(float2)) +
         static_cast<size_t>(chunk_grid()) * (sizeof(CutCell) + 2 * sizeof(int));
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
