// Products of groups of rows on the tensor cores (16-bit types), and the gradient of their matrices.
//
//   Y[r]  = X[r] * W[g]     accumulator tile: 128 columns of Y (lanes) x up to BN rows of one group (columns)
//   dW[g] = A_g^T * B_g     accumulator tile: 128 columns of dW (lanes) x up to BN rows of dW (columns)
//
// One warp issues TMA copies into a ring of swizzled tiles, one issues tcgen05.mma on them, four carry finished
// accumulators from tensor memory to global memory while the next tile is multiplied into the other half.  The matrix (W)
// sits on the 128-wide side of the instruction and the rows on its N side, which the instruction takes in steps of 16 up to
// 256: a tile costs as much as the rows that its group has, whether that is one row or 256, and a lane's neighbours hold
// neighbouring columns of Y, so that a warp's stores are contiguous.  Blocks stay for the whole call (one to an SM) and take
// tiles in turn; the tiles follow from the offsets, which only the device knows.  Bound by the tensor cores and, in a row of
// such calls, by the power they take: 32,768 rows of 8 groups, 2048 x 5632, bf16, alone 1.29 to 1.44 PFLOP/s; 16,384 rows of 32
// groups, 2048 x 2816, 1.1 alone and 0.9 in a row; a step of a decoder (56 rows in 64 groups, 2048 x 1536) by the bytes of the
// matrices: 6.2 TB/s.
// Large calls take tiles of 256 x 256 in pairs of blocks (cta_group::2).  Where the tiles are fewer than the SMs (a step of a
// decoder), clusters of 2 to 8 blocks split the depth of one tile and
// add their parts through distributed shared memory, in the order of their ranks.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "dense_types.cuh"
#include "device_utils.cuh"
#include "grouped.cuh"

namespace {

using namespace hpspmm;

constexpr int kThreads = 256;
constexpr int kLanes = 128;                    // columns of the output to a tile
constexpr int kDepth = 64;                     // of one stage: 128 bytes, the span of the swizzle
constexpr int kABytes = kLanes * kDepth * 2;
constexpr int kMaxGroups = kMostSplitGroups;   // of one launch: their tile counts lie in shared memory
constexpr int kMaxTiles = 0x7fff0000;          // of one launch: adding a grid to it stays within 31 bits
constexpr int kMostTiles = 1 << 29;            // where the sum of the groups' tiles stops: two of them are below 2^31

enum { MODE_OUT_FIRST, MODE_IN_FIRST, MODE_WEIGHT };   // W stored [G, N, K], [G, K, N]; gradient of the matrices

struct tensor_args {
  const int* offsets;
  int R, G;            // rows, groups of the call
  int g0, gn;          // groups of this launch
  int depth;           // products: K
  int rows, cols;      // of the output: products: -, N; gradients: rows and columns of one matrix
  int zero_rows;       // products: whether this launch clears the rows of no group
  piece_plan plan;     // gradients
  float* slots;
  int *timeouts, *alarm;   // counted and told where a wait was given up
  // the operands on the lanes and on the N side, for calls whose tiles TMA cannot fetch: rows ld elements apart
  const void *a, *b;
  int64_t lda, ldb;
  long long wait_limit;   // cycles, see wait_state
  int withhold;           // (for tests) nothing is copied, so that the waits for the copies run out
};

// ---- instructions ------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar, int rank) {
  asm volatile(
      "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n"
      " mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n}\n" ::"r"(bar), "r"(rank) : "memory");
}
// A wait may sleep that many nanoseconds in the hardware.  Without the hint six of the eight warps polled, which on a GPU at
// its power limit was taken from the products: 1979 us for what takes 1859 (32,768 rows of 8 groups, 2048 x 5632, with both
// gradients, over 1.5 s).
constexpr uint32_t kSleep = 1000000;

template <bool CLUSTER>
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  if (CLUSTER)
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(kSleep) : "memory");
  else
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(kSleep) : "memory");
  return ok != 0;
}
// What the waits of a block share.
struct wait_state {
  int failed;          // one of them has been given up, so all others are
  long long limit;     // cycles that one may take beside kStageLimit for every stage that comes in meanwhile
};
// A stage takes 0.3 us with TMA and 2.1 at most without (4,200 cycles); a tile has up to 2^21 of them.
constexpr long long kStageLimit = 20000;
// By one thread.  Whoever gives up says so in `failed`, and all others give up with it.
__device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, volatile wait_state* w) {
  const long long begin = clock64();
  while (true) {
    if (mbar_try<false>(bar, parity)) return true;
    if (w->failed) return false;
    if (clock64() - begin > w->limit) {
      w->failed = 1;
      return false;
    }
  }
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile wait_state* w) {
  return mbar_try<false>(bar, parity) || mbar_wait_slow(bar, parity, w);
}
// By a whole warp, with the same answer in all lanes: what follows are instructions that all of them have to reach, so that
// lanes which gave up while others did not would leave those waiting for good.  stages: how many may come in before the wait
// is over; a tile's for its accumulator.
template <bool CLUSTER>
__device__ __noinline__ bool mbar_wait_warp_slow(uint32_t bar, uint32_t parity, volatile wait_state* w, int stages) {
  const long long begin = clock64();
  while (true) {
    if (__all_sync(0xffffffffu, mbar_try<CLUSTER>(bar, parity))) return true;
    if (__any_sync(0xffffffffu, w->failed || clock64() - begin > w->limit + stages * kStageLimit)) {
      w->failed = 1;
      return false;
    }
  }
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile wait_state* w, int stages = 0) {
  return __all_sync(0xffffffffu, mbar_try<CLUSTER>(bar, parity)) || mbar_wait_warp_slow<CLUSTER>(bar, parity, w, stages);
}

// PAIR: the barrier may be the one of the pair's other block (`bar` is an address in the cluster's window)
template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if (PAIR)
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if (PAIR)
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
                 "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t in_block(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

// Shared-memory operand, 128-byte swizzle.  Along the depth (LINES_OF_DEPTH: every 128-byte line holds 64 elements along
// the depth): groups of 8 lines 1024 bytes apart.  Across it (a line holds 64 elements across the depth): 8 lines of depth
// 1024 bytes apart, the next 64 elements across 64 lines = 8192 bytes further.
template <bool LINES_OF_DEPTH>
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  const uint64_t lead = LINES_OF_DEPTH ? 1 : (kDepth * 128) >> 4;
  return (uint64_t)((addr & 0x3ffff) >> 4) | lead << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// 16 elements further along the depth, in the descriptor's units of 16 bytes
template <bool LINES_OF_DEPTH>
__device__ __forceinline__ constexpr uint64_t operand_step() { return LINES_OF_DEPTH ? 32 >> 4 : (16 * 128) >> 4; }

template <bool PAIR>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add) {
  if (PAIR)
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(instr), "r"((int)add) : "memory");
  else
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(instr), "r"((int)add) : "memory");
}
// arrives (in a pair: at both blocks' barrier of that place) once the products issued so far are done
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"((uint16_t)3) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
template <bool PAIR, int COLUMNS>
__device__ __forceinline__ void tensor_alloc(uint32_t to) {
  if (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "n"(COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(to), "n"(COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}
template <bool PAIR, int COLUMNS>
__device__ __forceinline__ void tensor_free(uint32_t base) {
  if (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLUMNS) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLUMNS) : "memory");
}
__device__ __forceinline__ void tensor_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of the warp's 32 lanes
__device__ __forceinline__ void tensor_load(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
      "%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
        "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
        "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// ---- tiles -------------------------------------------------------------------------------------------------------

struct tile {
  int g;               // group
  int row0, rows;      // of the output, inside Y or inside the group's matrix
  int col0;            // of the output
  int begin, end;      // depth: products: stages of this block; gradients: rows of the group
  int stages;
  int slot;            // gradients: where a piece of a group goes, -1: to the matrix itself
};

// WIDTH: columns of the output to a tile (128, of a pair of blocks 256)
template <int MODE, int BN, int WIDTH>
__device__ __forceinline__ int tile_count(const tensor_args& a, const int* ends) {
  const int across = (a.cols + WIDTH - 1) / WIDTH;
  if (MODE == MODE_WEIGHT)
    return (int)min((int64_t)(a.plan.slots ? ends[a.gn - 1] : a.gn) * ((a.rows + BN - 1) / BN) * across, (int64_t)kMaxTiles);
  return (int)min((int64_t)ends[a.gn - 1] * across, (int64_t)kMaxTiles);
}

template <int MODE, int BN, int CL, bool PAIR>
__device__ __forceinline__ tile tile_at(const tensor_args& a, const int* ends, const int* slot_ends, int u, int rank) {
  tile t;
  constexpr int kWidth = PAIR ? 2 * kLanes : kLanes;
  const int across = (a.cols + kWidth - 1) / kWidth;
  int q = u / across;
  t.col0 = (u - q * across) * kWidth + (PAIR ? rank * kLanes : 0);
  t.slot = -1;
  if (MODE == MODE_WEIGHT) {
    const int down = (a.rows + BN - 1) / BN;
    t.row0 = (q % down) * BN;
    q /= down;
    t.rows = min(BN, a.rows - t.row0);
  }
  int lo = 0, hi = a.gn - 1;
  if (MODE == MODE_WEIGHT && !a.plan.slots) {
    lo = q;
  } else {
    while (lo < hi) {
      const int m = (lo + hi) >> 1;
      if (ends[m] > q) hi = m; else lo = m + 1;
    }
  }
  t.g = a.g0 + lo;
  if (MODE == MODE_WEIGHT) {
    part_bounds(a.offsets, a.G, a.R, t.g, t.begin, t.end);
    if (a.plan.slots) {
      const int piece = q - (lo ? ends[lo - 1] : 0);
      if (pieces_of(max(t.end - t.begin, 0), a.plan.length) > 1) t.slot = (lo ? slot_ends[lo - 1] : 0) + piece;
      t.begin += piece * a.plan.length;
      t.end = t.begin + min(t.end - t.begin, a.plan.length);
    }
    t.stages = (max(t.end - t.begin, 0) + kDepth - 1) / kDepth;
    return t;
  }
  const int first = lo ? ends[lo - 1] : 0, tiles = ends[lo] - first;
  int begin, end;
  part_bounds(a.offsets, a.G, a.R, t.g, begin, end);
  // equal tiles, in steps of the instruction's 16; never more than BN rows, and as tiles = ceil(rows / BN), none is empty
  // (offsets that do not ascend can have more rows than there are, and their count of tiles is cut off)
  const int step = min(((end - begin - 1) / tiles + 16) / 16 * 16, BN);
  t.row0 = begin + (q - first) * step;
  t.rows = min(step, end - t.row0);
  const int stages = (a.depth + kDepth - 1) / kDepth;
  t.begin = CL == 1 ? 0 : (int)((int64_t)stages * rank / CL);
  t.end = CL == 1 ? stages : (int)((int64_t)stages * (rank + 1) / CL);
  t.stages = t.end - t.begin;
  return t;
}

// Whether a stage of a gradient ends inside the instruction's depth of 16: the rows behind belong to the next group.
__device__ __forceinline__ bool cut_short(const tile& t, int stage) {
  const int left = t.end - t.begin - stage * kDepth;
  return left < kDepth && (left & 15);
}

template <typename T>
struct type_code;
template <>
struct type_code<__half> { static constexpr uint32_t value = 0; };
template <>
struct type_code<__nv_bfloat16> { static constexpr uint32_t value = 1; };

// ---- tiles without TMA ---------------------------------------------------------------------------------------------
//
// Operands whose rows do not begin on 16-byte boundaries: eight warps bring a tile in, two such teams in turn, 128 bytes of
// neighbouring elements to a warp, two to a lane, and write it swizzled as TMA does.  Loads go without a branch, from an element that is
// there where the wanted one is not: conditional loads of one batch waited for one another, 0.7 us each.  (Aligned words,
// shifted by half a word where a row begins in the middle of one, took a third of the loads and ten times the
// instructions: 78 us where this takes 22.9, for 5,003 rows of 13 groups, 333 x 131.)

constexpr int kLoaders = 8;     // warps of a team
constexpr int kTeams = 2;
constexpr int kLinesInFlight = 16;

// Lines `warp`, `warp` + kLoaders, ... of an operand's tile.  Line i holds 64 elements of row `row + i % PER` (there is none
// from `rows` on) from column `col + 64 * (i / PER)` (there is none from `cols` on): zeros stand for what is not there.
template <int PER>
__device__ __forceinline__ void load_lines(const uint16_t* p, int64_t ld, int warp, int lines, int64_t row, int64_t rows, int col, int cols,
                                           uint32_t tile) {
  const int lane = threadIdx.x & 31, present = (int)min(rows - row, (int64_t)PER);
  for (int first = 0; first < lines; first += PER) {
    const int c = col + 64 * (first / PER), valid = min(max(cols - c, 0), 64), n = min(PER, lines - first);
    // the lane's elements, and which of them count
    const int e0 = min(2 * lane, valid - 1), e1 = min(2 * lane + 1, valid - 1);
    const uint32_t keep = (2 * lane < valid ? 0xffffu : 0u) | (2 * lane + 1 < valid ? 0xffff0000u : 0u);
    const uint16_t* from = p + row * ld + c;
    for (int i0 = warp; i0 < n; i0 += kLoaders * kLinesInFlight) {
      uint32_t low[kLinesInFlight], high[kLinesInFlight];
#pragma unroll
      for (int j = 0; j < kLinesInFlight; ++j) low[j] = high[j] = 0;
      if (valid > 0) {
#pragma unroll
        for (int j = 0; j < kLinesInFlight; ++j) {
          const uint16_t* at = from + min(i0 + j * kLoaders, present - 1) * ld;
          low[j] = __ldg(at + e0), high[j] = __ldg(at + e1);
        }
      }
#pragma unroll
      for (int j = 0; j < kLinesInFlight; ++j) {
        const int i = i0 + j * kLoaders;
        if (i < n) {
          const uint32_t v = i < present ? (low[j] | high[j] << 16) & keep : 0;
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(tile + (first + i) * 128 + (((lane >> 2) ^ (i & 7)) << 4) + (lane & 3) * 4), "r"(v)
                       : "memory");
        }
      }
    }
  }
}

template <int BN, int STAGES, int CL, bool PAIR>
constexpr int smem_bytes() { return 1024 + STAGES * (kABytes + BN * 128 / (PAIR ? 2 : 1)) + (CL > 1 ? BN * kLanes * 4 : 0); }

template <typename T, int MODE, int BN, int STAGES, int CL, bool TMA, bool PAIR>
__global__ void __launch_bounds__(TMA ? kThreads : kThreads + kTeams * kLoaders * 32, 1)
grouped_tensor_kernel(const tensor_args a, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                      T* __restrict__ out) {
  constexpr bool kWeight = MODE == MODE_WEIGHT;
  constexpr bool kALines = MODE == MODE_OUT_FIRST, kBLines = !kWeight;   // which operands have lines along the depth
  constexpr int kBlocks = PAIR ? 2 : CL;                                 // of a cluster
  static_assert(!PAIR || (CL == 1 && TMA), "pairs neither split the depth nor go without TMA");
  // of the N side, a block of a pair holds one half
  constexpr int kBBytes = BN * 128 / (PAIR ? 2 : 1), kStage = kABytes + kBBytes;
  constexpr int kColumns = 2 * BN < 32 ? 32 : 2 * BN;                   // of tensor memory: two accumulators
  extern __shared__ char raw[];
  __shared__ int ends[kMaxGroups];
  __shared__ int slot_ends[kWeight ? kMaxGroups : 1];
  __shared__ int part[kThreads / 32];
  __shared__ uint64_t bars[4 * STAGES + 6];
  __shared__ uint32_t tmem_base;
  __shared__ wait_state waits;
  const uint32_t base = (smem_of(raw) + 1023) / 1024 * 1024;
  const uint32_t bar0 = smem_of(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto acc_full = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  auto acc_empty = [&](int b) { return bar0 + 8u * (2 * STAGES + 2 + b); };
  auto cut_full = [&](int s) { return bar0 + 8u * (3 * STAGES + 6 + s); };  // a stage that is cut short has been copied
  auto cleared = [&](int s) { return bar0 + 8u * (2 * STAGES + 6 + s); };   // and has its zeros
  const uint32_t parts_full = bar0 + 8u * (2 * STAGES + 4), parts_empty = bar0 + 8u * (2 * STAGES + 5);
  float* const parts = reinterpret_cast<float*>(raw + (base - smem_of(raw)) + STAGES * kStage);   // [source][row][lane]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int rank = 0;
  if (kBlocks > 1) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));

  if (threadIdx.x == 0) {
    waits.failed = 0, waits.limit = a.wait_limit;
    for (int s = 0; s < STAGES; ++s) mbar_init(full(s), TMA ? 1 : kLoaders), mbar_init(empty(s), 1), mbar_init(cleared(s), PAIR ? 2 : 1), mbar_init(cut_full(s), 1);
    for (int b = 0; b < 2; ++b) mbar_init(acc_full(b), 1), mbar_init(acc_empty(b), PAIR ? 8 : 4);
    mbar_init(parts_full, 4 * CL), mbar_init(parts_empty, 4 * CL);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (TMA) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
    }
  }
  if (warp == 2) {
    tensor_alloc<PAIR, kColumns>(smem_of(&tmem_base));
    tensor_fence_before();
  }
  chain_grid();

  // How many tiles (pieces) the groups up to each one have, and how many slots
  auto prefix = [&](int* to, bool slots) {
    constexpr int kPer = kMaxGroups / kThreads;
    const bool counts = TMA || threadIdx.x < kThreads;
    int n[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = counts ? threadIdx.x * kPer + i : a.gn;
      int begin = 0, end = 0;
      if (g < a.gn) part_bounds(a.offsets, a.G, a.R, a.g0 + g, begin, end);
      const int rows = max(end - begin, 0);
      if (!kWeight)
        n[i] = (rows + BN - 1) / BN;
      else
        n[i] = g < a.gn ? pieces_of(rows, a.plan.length) : 0;
      if (slots && n[i] < 2) n[i] = 0;
      sum = min(sum + n[i], kMostTiles);
    }
    int before = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before = min(before + o, kMostTiles);
    }
    if (counts && lane == 31) part[warp] = before;
    __syncthreads();
    before = max(before - sum, 0);
    if (counts) {
      for (int w = 0; w < warp; ++w) before = min(before + part[w], kMostTiles);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        before = min(before + n[i], kMostTiles);
        to[threadIdx.x * kPer + i] = before;
      }
    }
    __syncthreads();
  };
  if (!kWeight || a.plan.slots) prefix(ends, false);
  if (kWeight && a.plan.slots) prefix(slot_ends, true);
  __syncthreads();
  // The others' barriers are ready: a pair needs them from the first copy on, blocks that split the depth only when they join
  // their parts, and whoever does not waits at the end.
  if (kBlocks > 1) cluster_arrive();
  if (PAIR) cluster_wait();
  tensor_fence_after();
  const uint32_t tmem = tmem_base;
  const int units = tile_count<MODE, BN, PAIR ? 2 * kLanes : kLanes>(a, ends);
  const int first = blockIdx.x / kBlocks, step = gridDim.x / kBlocks;

  if (warp == 0) {
    if (TMA && lane == 0 && !a.withhold) {   // copies
      int s = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int u = first; u < units && ok; u += step) {
        const tile t = tile_at<MODE, BN, CL, PAIR>(a, ends, slot_ends, u, rank);
        // of the N side, this block's part: rows [from, from + count)
        const int half = (t.rows + 31) / 32 * 16;
        const int from = t.row0 + (PAIR ? rank * half : 0), count = PAIR ? half : t.rows;
        const int boxes = (count + 63) / 64;
        for (int k = 0; k < t.stages; ++k) {
          ok = mbar_wait(empty(s), phase ^ 1, &waits);
          if (!ok) break;
          // The copies of both blocks of a pair arrive at the first one's barrier.  A stage that is cut short has a barrier of
          // its own, in either block: its rest has to be cleared before it is used.
          const bool cut = kWeight && cut_short(t, k), shared = PAIR && !cut;
          const uint32_t dst = base + s * kStage, own = cut ? cut_full(s) : full(s), bar = shared ? in_block(own, 0) : own;
          const uint32_t bytes = kABytes + boxes * 8192;
          if (!shared || rank == 0) mbar_expect(own, shared ? 2 * bytes : bytes);
          if (kWeight) {
            const int r = t.begin + k * kDepth;
            tma_load<PAIR>(dst, &map_a, bar, t.col0, r);
            tma_load<PAIR>(dst + 8192, &map_a, bar, t.col0 + 64, r);
            for (int b = 0; b < boxes; ++b) tma_load<PAIR>(dst + kABytes + b * 8192, &map_b, bar, from + b * 64, r);
          } else {
            const int d = (t.begin + k) * kDepth;
            if (MODE == MODE_OUT_FIRST) {
              tma_load<PAIR>(dst, &map_a, bar, d, t.col0, t.g);
            } else {
              tma_load<PAIR>(dst, &map_a, bar, t.col0, d, t.g);
              tma_load<PAIR>(dst + 8192, &map_a, bar, t.col0 + 64, d, t.g);
            }
            for (int b = 0; b < boxes; ++b) tma_load<PAIR>(dst + kABytes + b * 8192, &map_b, bar, d, from + b * 64);
          }
          if (++s == STAGES) s = 0, phase ^= 1;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // Products, by one thread (of a pair: the first block's).  The next instruction has to be there when the one before it
    // ends, 128 cycles later.  With the next tile looked up between two tiles the tensor cores stood still for a third of the
    // time; a look at the next stage's barrier between two products of one cost 10 %; and the warp stays together, so that
    // descriptors are kept in uniform registers: 3 % ahead of one lane on its own.
    if (!(PAIR && rank)) {
      uint32_t one;
      asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
      struct {
        int stages, rows, steps;   // steps: of 16 of the depth, in the last stage
        bool cut;
      } w, next = {};
      auto look_up = [&](int u) {
        if (u >= units) return;
        const tile t = tile_at<MODE, BN, CL, PAIR>(a, ends, slot_ends, u, rank);
        const int left = (kWeight ? t.end - t.begin : a.depth - t.begin * kDepth) - (t.stages - 1) * kDepth;
        next.stages = t.stages, next.rows = t.rows, next.steps = min(kDepth / 16, (left + 15) / 16);
        next.cut = kWeight && TMA && t.stages > 0 && cut_short(t, t.stages - 1);
        // (the same in all lanes, and known to be)
        next.stages = __shfl_sync(0xffffffffu, next.stages, 0), next.rows = __shfl_sync(0xffffffffu, next.rows, 0);
        next.steps = __shfl_sync(0xffffffffu, next.steps, 0), next.cut = __shfl_sync(0xffffffffu, (int)next.cut, 0);
      };
      const uint64_t first_a = operand<kALines>(base), first_b = operand<kBLines>(base + kABytes);
      int s = 0, acc = 0;
      uint32_t acc_phase = 0, full_phase = 0, cut_phase = 0;   // a bit for each stage, which has two barriers
      bool ok = true;
      look_up(first);
      for (int u = first; u < units && ok; u += step) {
        w = next;
        ok = mbar_wait_warp<PAIR>(acc_empty(acc), acc_phase ^ 1, &waits);
        if (!ok) break;
        tensor_fence_after();
        const uint32_t d = tmem + acc * BN;
        const int n = PAIR ? (w.rows + 31) / 32 * 32 : (w.rows + 15) / 16 * 16;
        // accumulate in 32 bits; type of A and B; whether their lines run across the depth; N / 8; M / 16
        const uint32_t instr = 1u << 4 | type_code<T>::value << 7 | type_code<T>::value << 10 | (uint32_t)!kALines << 15 |
                               (uint32_t)!kBLines << 16 | (uint32_t)(n >> 3) << 17 | (uint32_t)((PAIR ? 2 : 1) * kLanes >> 4) << 24;
        for (int k = 0; k < w.stages; ++k) {
          const bool last = k + 1 == w.stages;
          if (last && w.cut) {
            ok = mbar_wait_warp<PAIR>(cleared(s), cut_phase >> s & 1, &waits);
            cut_phase ^= 1u << s;
          } else {
            ok = mbar_wait_warp(full(s), full_phase >> s & 1, &waits);
            full_phase ^= 1u << s;
          }
          if (!ok) break;
          tensor_fence_after();
          const uint64_t da = first_a + (uint64_t)(s * (kStage >> 4)), db = first_b + (uint64_t)(s * (kStage >> 4));
          const int steps = last ? w.steps : kDepth / 16;
          if (one) {
            mma<PAIR>(d, da, db, instr, k > 0);
#pragma unroll
            for (int i = 1; i < kDepth / 16; ++i)
              if (i < steps) mma<PAIR>(d, da + i * operand_step<kALines>(), db + i * operand_step<kBLines>(), instr, true);
            mma_commit<PAIR>(empty(s));
          }
          __syncwarp();
          if (k == 0) look_up(u + step);
          if (++s == STAGES) s = 0;
        }
        if (!ok) break;
        if (w.stages == 0) look_up(u + step);
        if (one) {
          if (w.stages) {
            mma_commit<PAIR>(acc_full(acc));
          } else {
            mbar_arrive(acc_full(acc));
            if (PAIR) mbar_arrive_remote(acc_full(acc), 1);
          }
        }
        __syncwarp();
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
    }
    __syncwarp();
  } else if (kWeight && TMA && warp == 3) {   // the rows behind a group, up to the end of the instruction's depth, become zeros
    int s = 0;
    uint32_t phase = 0;   // a bit for each stage
    int stages = 0;       // since the last one that was cut short
    for (int u = first; u < units; u += step) {
      const tile t = tile_at<MODE, BN, CL, PAIR>(a, ends, slot_ends, u, rank);
      if (t.stages == 0) continue;
      s = (s + t.stages - 1) % STAGES;
      stages = min(stages + t.stages, 1 << 30);
      if (cut_short(t, t.stages - 1)) {
        if (!mbar_wait_warp(cut_full(s), phase >> s & 1, &waits, stages)) break;
        stages = 0;
        phase ^= 1u << s;
        const uint32_t src = base + s * kStage;
        const int left = t.end - t.begin - (t.stages - 1) * kDepth;
        const int wide = 2 + ((PAIR ? (t.rows + 31) / 32 * 16 : t.rows) + 63) / 64, rows = 16 - (left & 15);
        for (int i = lane; i < wide * rows * 8; i += 32) {
          const int b = i / (rows * 8), r = left + (i >> 3) % rows;
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(src + b * 8192 + r * 128 + (i & 7) * 16), "r"(0) : "memory");
        }
        asm volatile("fence.proxy.async;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_remote(cleared(s), 0); else mbar_arrive(cleared(s));
        }
        __syncwarp();
      }
      s = (s + 1) % STAGES;
    }
  } else if (!TMA && warp >= kThreads / 32) {   // copies, line by line
    const int w = (warp - kThreads / 32) % kLoaders, team = (warp - kThreads / 32) / kLoaders;
    const uint16_t *pa = static_cast<const uint16_t*>(a.a), *pb = static_cast<const uint16_t*>(a.b);
    int s = 0, turn = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int u = a.withhold ? units : first; u < units && ok; u += step) {
      const tile t = tile_at<MODE, BN, CL, PAIR>(a, ends, slot_ends, u, rank);
      for (int k = 0; k < t.stages; ++k) {
        const int at = s;
        const uint32_t parity = phase ^ 1;
        if (++s == STAGES) s = 0, phase ^= 1;
        turn = turn + 1 == kTeams ? 0 : turn + 1;
        if (turn != team) continue;
        ok = mbar_wait_warp(empty(at), parity, &waits);
        if (!ok) break;
        const uint32_t dst = base + at * kStage;
        if (kWeight) {
          const int64_t r = (int64_t)t.begin + k * kDepth;
          load_lines<kDepth>(pa, a.lda, w, kLanes, r, t.end, t.col0, a.cols, dst);
          load_lines<kDepth>(pb, a.ldb, w, (t.rows + 63) / 64 * kDepth, r, t.end, t.row0, a.rows, dst + kABytes);
        } else {
          const int d = (t.begin + k) * kDepth;
          const uint16_t* wg = pa + (int64_t)t.g * a.depth * a.cols;
          if (MODE == MODE_OUT_FIRST)
            load_lines<kLanes>(wg, a.lda, w, kLanes, t.col0, a.cols, d, a.depth, dst);
          else
            load_lines<kDepth>(wg, a.lda, w, kLanes, d, a.depth, t.col0, a.cols, dst);
          load_lines<BN>(pb, a.ldb, w, t.rows, t.row0, a.R, d, a.depth, dst + kABytes);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(full(at));
      }
    }
  } else if (warp >= 4) {   // results
    const int q = warp - 4;
    auto acc_left = [&](int b) {   // whoever issues the products may write it again
      if (PAIR) mbar_arrive_remote(acc_empty(b), 0); else mbar_arrive(acc_empty(b));
    };
    int acc = 0;
    uint32_t acc_phase = 0, part_phase = 0;
    if (CL > 1) cluster_wait();
    for (int u = first; u < units; u += step) {
      const tile t = tile_at<MODE, BN, CL, PAIR>(a, ends, slot_ends, u, rank);
      if (!mbar_wait_warp(acc_full(acc), acc_phase, &waits, t.stages)) break;
      tensor_fence_after();
      const uint32_t src = tmem + acc * BN + ((uint32_t)(q * 32) << 16);
      const int col = t.col0 + q * 32 + lane;
      const bool inside = col < a.cols;
      T* to = out + (kWeight ? (int64_t)t.g * a.rows * a.cols : 0) + (int64_t)t.row0 * a.cols + col;
      if (kWeight && t.slot >= 0) {   // a piece of a group, in 32 bits
        float* piece = a.slots + (int64_t)t.slot * a.rows * a.cols + (int64_t)t.row0 * a.cols + col;
        for (int c = 0; c < t.rows; c += 32) {
          uint32_t v[32];
          tensor_load(src + c, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (inside && c + j < t.rows && t.slot < a.plan.slots) *piece = __uint_as_float(v[j]);
            piece += a.cols;
          }
        }
        tensor_fence_before();
        __syncwarp();
        if (lane == 0) acc_left(acc);
      } else if (CL == 1) {
        for (int c = 0; c < t.rows; c += 32) {
          uint32_t v[32];
          tensor_load(src + c, v);
          if (kWeight && t.stages == 0) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0;
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (inside && c + j < t.rows) *to = from_float<T>(__uint_as_float(v[j]));
            to += a.cols;
          }
        }
        tensor_fence_before();
        __syncwarp();
        if (lane == 0) acc_left(acc);
      } else {
        // Every block takes 1 / CL of the tile's rows and gets the others' parts of them pushed into its shared memory.
        const int share = (t.rows + 15) / 16 * 16 / CL;
        if (!mbar_wait_warp<true>(parts_empty, part_phase ^ 1, &waits, t.stages)) break;
        const uint32_t mine = smem_of(parts + rank * share * kLanes + q * 32 + lane);
        int to_rank = 0, r = 0;
        uint32_t at = in_block(mine, 0);
        for (int c = 0; c < CL * share; c += 32) {
          uint32_t v[32];
          tensor_load(src + c, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            if (c + j < CL * share) {
              asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(v[j]) : "memory");
              at += kLanes * 4;
              if (++r == share) {
                r = 0, ++to_rank;
                if (to_rank < CL) at = in_block(mine, to_rank);
              }
            }
          }
        }
        tensor_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(acc_empty(acc));
          for (int p = 0; p < CL; ++p) mbar_arrive_remote(parts_full, p);
        }
        __syncwarp();
        if (!mbar_wait_warp<true>(parts_full, part_phase, &waits, t.stages)) break;
        for (int r = 0; r < share; ++r) {
          float sum = 0.f;
#pragma unroll
          for (int p = 0; p < CL; ++p) sum += parts[(p * share + r) * kLanes + q * 32 + lane];
          const int row = rank * share + r;
          if (inside && row < t.rows) to[(int64_t)row * a.cols] = from_float<T>(sum);
        }
        __syncwarp();
        if (lane == 0)
          for (int p = 0; p < CL; ++p) mbar_arrive_remote(parts_empty, p);
        part_phase ^= 1;
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  } else if (!kWeight && a.zero_rows && (warp == 2 || warp == 3)) {   // rows of no group, by the two warps that are left
    typedef typename raw_bytes<TMA ? 16 : 2>::type word;
    const int64_t width = TMA ? a.cols / 8 : a.cols;     // words to a row
    word* words = reinterpret_cast<word*>(out);
    const int64_t at = (int64_t)blockIdx.x * 64 + (threadIdx.x - 64), all = (int64_t)gridDim.x * 64;
    for (int i = a.G; i < a.G + 2; ++i) {
      int begin, end;
      part_bounds(a.offsets, a.G, a.R, i, begin, end);
      for (int64_t w = begin * width + at; w < end * width; w += all) words[w] = word{};
    }
  }
  tensor_fence_before();
  __syncthreads();
  if (waits.failed) {   // what was started lands before the memory is given back
    if (threadIdx.x == 0) {
      atomicAdd(a.timeouts, 1);
      *static_cast<volatile int*>(a.alarm) = 1;
      __threadfence_system();
    }
    const long long begin = clock64();
    while (clock64() - begin < 4000000ll) __nanosleep(1000);
    __syncwarp();
  }
  if (kBlocks > 1) {   // nobody reaches into the memory of a block that has left
    if (CL > 1 && (warp < 4 || warp >= kThreads / 32)) cluster_wait();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 2) {
    tensor_fence_after();
    tensor_free<PAIR, kColumns>(tmem);
  }
}

// ---- launches -----------------------------------------------------------------------------------------------------

// Of a wait, in cycles: about two seconds (and kStageLimit for a stage).  hpspmm_debug_grouped_waits changes it, and withholds
// the copies.
constexpr int64_t kWaitLimit = 4000000000ll;
std::atomic<int64_t> g_wait_limit{kWaitLimit};
std::atomic<int> g_withhold{0};

typedef CUresult (*encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A dense array of 16-bit elements, innermost dimension first; strides in elements of all but the innermost.
bool encode(CUtensorMap* map, bool half, const void* p, int dims, const int64_t* size, const int64_t* stride, const int* box) {
  encode_fn fn = (encode_fn)hpspmm_tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t sizes[3], strides[2];
  cuuint32_t boxes[3], ones[3] = {1, 1, 1};
  for (int i = 0; i < dims; ++i) sizes[i] = (cuuint64_t)size[i], boxes[i] = (cuuint32_t)box[i];
  for (int i = 0; i + 1 < dims; ++i) {
    if (stride[i] >= (int64_t)1 << 38) return false;
    strides[i] = (cuuint64_t)stride[i] * 2;
  }
  return fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dims, const_cast<void*>(p), sizes, strides,
            boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int MODE, int BN, int STAGES, int CL, bool TMA, bool PAIR = false>
cudaError_t launch_one(hpspmm_ctx* ctx, const tensor_args& a, const CUtensorMap& ma, const CUtensorMap& mb, void* out, int64_t units,
                       cudaStream_t s) {
  auto* kernel = grouped_tensor_kernel<T, MODE, BN, STAGES, CL, TMA, PAIR>;
  constexpr int smem = smem_bytes<BN, STAGES, CL, PAIR>();
  // per call: the attribute belongs to the current device's context, and a process may drive several GPUs
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  constexpr int kBlocks = PAIR ? 2 : CL;
  attr[1].val.clusterDim.x = kBlocks, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3((unsigned)(std::min<int64_t>(units, ctx->sm_count / kBlocks) * kBlocks));
  c.blockDim = dim3(TMA ? kThreads : kThreads + kTeams * kLoaders * 32);
  c.dynamicSmemBytes = smem, c.stream = s, c.attrs = attr, c.numAttrs = kBlocks > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&c, kernel, a, ma, mb, (T*)out);
  ctx->launches++;
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Rows (of dW: rows of the output) to a tile, whether pairs of blocks take it, and how many blocks split its depth.
struct tile_choice {
  int rows;
  bool pair;
  int blocks;
};

// Two blocks to a tile of 256 x 256: each fetches one half of either operand, 64 bytes for every 128 x 128 x 1 products where
// a block alone fetches 96.  Where the output is wide enough that its last tile of 256 columns is not often half empty.
bool wide_enough_for_pairs(int64_t cols) { return cols > kLanes && (cols >= 1024 || (cols - 1) % 256 >= 128); }

// The choice for a product, from what was measured for a block's tile of 64, 128 or 256 rows and a pair's of 256 (1,024 to
// 5,632 wide, depth 64 to 4,096, 8 to 30,000 rows of 1 to 64 groups): `stage` us for 64 of the depth, `rest` for the tile,
// and not less than `store`, its way to memory.  The host does not know the groups' sizes: half a tile more than the rows
// need for each of them is assumed.  1,500 rows of one group, 2048 x 2048: 44 us with tiles of 64, 27 with 128, 19 with 256,
// 18 with pairs; 600 rows 22 / 16 / 18 / 17; 30,000 rows, 64 x 4096: 110 / 91 / 72 / 96.
// Splitting the depth costs 3 us and more, as long as all clusters run at once: 8 rows, 4096 x 1024: 20 us -> 11.5 with
// eight blocks; 1024 x 1024: 7.9 -> 9.8.
struct tile_cost {
  int rows;
  bool pair;
  double stage, rest, store;
};
constexpr tile_cost kTmaCosts[4] = {{64, false, 0.275, 0.7, 1.3}, {128, false, 0.40, 0.9, 1.8}, {256, false, 0.47, 1.6, 2.8},
                                    {256, true, 0.43, 1.6, 4.2}};
constexpr tile_cost kLineCosts[3] = {{64, false, 1.45, 0.7, 1.3}, {128, false, 1.65, 0.9, 1.8}, {256, false, 2.1, 1.6, 2.8}};
constexpr int kMostClusters[4] = {148, 72, 32, 12};   // of 1, 2, 4, 8 blocks, that are sure to run at once

tile_choice choose_product(int64_t R, int64_t G, int64_t K, int64_t cols, bool tma) {
  const double stages = (double)((K + kDepth - 1) / kDepth), groups = (double)std::min(R, G);
  tile_choice best = {64, false, 1};
  double least = 1e30;
  for (int i = 0; i < (tma ? 4 : 3); ++i) {
    const tile_cost& c = tma ? kTmaCosts[i] : kLineCosts[i];
    if (c.pair && !wide_enough_for_pairs(cols)) continue;
    const double width = c.pair ? 2 * kLanes : kLanes, across = std::ceil((double)cols / width);
    const double tiles = across * std::max(groups, (double)R / c.rows + groups / 2);
    const double t = std::ceil(tiles / (c.pair ? 74 : 148)) * std::max(c.store, stages * c.stage + c.rest);
    if (t < least) best = {c.rows, c.pair, 1}, least = t;
    for (int n = 1; i == 0 && n < 4 && stages >= 2 << n; ++n) {   // at least two stages to a block
      const double split = stages / (1 << n) * c.stage + c.rest + 3 + 0.4 * n;
      if (tiles <= kMostClusters[n] && split < least) best = {c.rows, false, 1 << n}, least = split;
    }
  }
  return best;
}

// The choice for a gradient, whose depth is the rows of a group (or of a piece of one).  Tiles enough for the SMs: 256 rows,
// pairs where there are about 512 rows to work on, below which a tile is little more than its stores (64 groups, 2048 x
// 2048: 189 us against 229 for 6,000 rows; 4 groups of 750: 37 against 36).  Fewer tiles: smaller ones (one group of 600
// rows, 1024 x 1024: 10.4 / 8.4 / 7.1 us with 256 / 128 / 64), and no larger than the output.  Without TMA 128 for twice as
// many whole groups (30,000 rows of 4 groups, 1025 x 1023: 672 / 512 / 746 us with 64 / 128 / 256).
tile_choice choose_gradient(int64_t R, int64_t G, int64_t I, int64_t J, const piece_plan& p, bool tma) {
  const double pieces = (double)G + p.slots / 2;   // (about half of the slots are used)
  const double tiles = pieces * (double)((I + 255) / 256) * (double)((J + kLanes - 1) / kLanes);
  if (tiles < 50 || I <= 64) return {64, false, 1};
  if (tiles < 100 || I <= 128 || (!tma && tiles < 200 && p.slots == 0)) return {128, false, 1};
  return {256, wide_enough_for_pairs(J) && (double)R / pieces >= 512, 1};
}

// What a product is launched with.
struct product_call {
  tensor_args a;
  CUtensorMap ma, mb;
  void* out;
  tile_choice tile;
  bool tma;
  int64_t units;   // no more tiles than that
};

template <typename T, int MODE, bool TMA>
cudaError_t launch_product(hpspmm_ctx* ctx, const product_call& c, cudaStream_t s) {
  if (TMA && c.tile.pair) return launch_one<T, MODE, 256, 6, 1, true, true>(ctx, c.a, c.ma, c.mb, c.out, c.units, s);
  if (c.tile.rows == 256) return launch_one<T, MODE, 256, 4, 1, TMA>(ctx, c.a, c.ma, c.mb, c.out, c.units, s);
  if (c.tile.rows == 128) return launch_one<T, MODE, 128, 6, 1, TMA>(ctx, c.a, c.ma, c.mb, c.out, c.units, s);
  if (c.tile.blocks == 8) return launch_one<T, MODE, 64, 7, 8, TMA>(ctx, c.a, c.ma, c.mb, c.out, c.units, s);
  if (c.tile.blocks == 4) return launch_one<T, MODE, 64, 7, 4, TMA>(ctx, c.a, c.ma, c.mb, c.out, c.units, s);
  if (c.tile.blocks == 2) return launch_one<T, MODE, 64, 7, 2, TMA>(ctx, c.a, c.ma, c.mb, c.out, c.units, s);
  return launch_one<T, MODE, 64, 8, 1, TMA>(ctx, c.a, c.ma, c.mb, c.out, c.units, s);
}
template <typename T>
cudaError_t launch_product(hpspmm_ctx* ctx, const product_call& c, bool out_first, cudaStream_t s) {
  if (c.tma)
    return out_first ? launch_product<T, MODE_OUT_FIRST, true>(ctx, c, s) : launch_product<T, MODE_IN_FIRST, true>(ctx, c, s);
  return out_first ? launch_product<T, MODE_OUT_FIRST, false>(ctx, c, s) : launch_product<T, MODE_IN_FIRST, false>(ctx, c, s);
}

template <typename T, bool TMA>
cudaError_t launch_weight_grad(hpspmm_ctx* ctx, const tensor_args& a, const CUtensorMap& ma, const CUtensorMap& mb, void* dW,
                               const tile_choice& c, int64_t units, cudaStream_t s) {
  if (TMA && c.pair) return launch_one<T, MODE_WEIGHT, 256, 6, 1, true, true>(ctx, a, ma, mb, dW, units, s);
  if (c.rows == 256) return launch_one<T, MODE_WEIGHT, 256, 4, 1, TMA>(ctx, a, ma, mb, dW, units, s);
  if (c.rows == 128) return launch_one<T, MODE_WEIGHT, 128, 6, 1, TMA>(ctx, a, ma, mb, dW, units, s);
  return launch_one<T, MODE_WEIGHT, 64, 8, 1, TMA>(ctx, a, ma, mb, dW, units, s);
}

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" int hpspmm_debug_grouped_waits(int64_t cycles, int32_t withhold) {
  if (cycles < 0) return HPSPMM_ERR_INVALID;
  g_wait_limit.store(cycles > 0 ? cycles : kWaitLimit, std::memory_order_relaxed);
  g_withhold.store(withhold != 0, std::memory_order_relaxed);
  return HPSPMM_OK;
}

int hpspmm_grouped_product_tensor(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t K, int64_t N, int32_t type, const void* X, int64_t ldx,
                                  const void* W, bool out_first, const int32_t* offsets, void* Y, cudaStream_t s) {
  const bool half = type == HPSPMM_TYPE_F16;
  product_call c = {};
  c.out = Y;
  const int64_t across = (N + kLanes - 1) / kLanes;
  if ((R / 64 + G + 1) * across > kMaxTiles || R / 64 + G + 1 > kMostTiles) return hpspmm_unsupported(ctx, "more than 2^31 tiles");
  const int64_t wsize[3] = {out_first ? K : N, out_first ? N : K, G}, wstride[2] = {wsize[0], K * N};
  const int wbox[3] = {64, out_first ? kLanes : kDepth, 1};
  const int64_t xsize[2] = {K, R}, xstride[1] = {ldx};
  const int xbox[2] = {kDepth, 64};
  c.tma = K % 8 == 0 && N % 8 == 0 && ldx % 8 == 0 && ldx >= K && aligned(X) && aligned(W) && aligned(Y) &&
          encode(&c.ma, half, W, 3, wsize, wstride, wbox) && encode(&c.mb, half, X, 2, xsize, xstride, xbox);
  c.tile = choose_product(R, G, K, N, c.tma);
  for (int64_t g0 = 0; g0 < G; g0 += kMaxGroups) {
    const int64_t gn = std::min<int64_t>(kMaxGroups, G - g0);
    c.a = {offsets, (int)R, (int)G, (int)g0, (int)gn, (int)K, 0, (int)N, g0 == 0, {(int)R, 0}, nullptr,
           ctx->flag + HPSPMM_FLAG_TENSOR_TIMEOUTS, ctx->alarm_dev, W, X, wsize[0], ldx,
           g_wait_limit.load(std::memory_order_relaxed), g_withhold.load(std::memory_order_relaxed)};
    c.units = (std::min(R, gn) + R / c.tile.rows) * across;
    HPSPMM_CUDA_TRY(ctx, half ? launch_product<__half>(ctx, c, out_first, s) : launch_product<__nv_bfloat16>(ctx, c, out_first, s));
  }
  return HPSPMM_OK;
}

// dW[g] (I x J) = A_g^T * B_g with A R x I and B R x J
int hpspmm_grouped_weight_grad_tensor(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t I, int64_t J, int32_t type, const void* A,
                                      int64_t lda, const void* B, int64_t ldb, const int32_t* offsets, void* dW,
                                      const piece_plan& p, float* slots, cudaStream_t s) {
  const bool half = type == HPSPMM_TYPE_F16;
  CUtensorMap ma = {}, mb = {};   // the operand of the output's columns lies on the lanes
  const int64_t asize[2] = {J, R}, astride[1] = {ldb}, bsize[2] = {I, R}, bstride[1] = {lda};
  const int box[2] = {64, kDepth};
  const bool tma = I % 8 == 0 && J % 8 == 0 && lda % 8 == 0 && ldb % 8 == 0 && lda >= I && ldb >= J && aligned(A) && aligned(B) &&
                   encode(&ma, half, B, 2, asize, astride, box) && encode(&mb, half, A, 2, bsize, bstride, box);
  const tile_choice c = choose_gradient(R, G, I, J, p, tma);
  const int64_t units = (G + p.slots) * ((I + c.rows - 1) / c.rows) * ((J + kLanes - 1) / kLanes);
  if (units > kMaxTiles) return hpspmm_unsupported(ctx, "more than 2^31 tiles");
  const tensor_args a = {offsets, (int)R, (int)G, 0, (int)G, 0, (int)I, (int)J, 0, p, slots, ctx->flag + HPSPMM_FLAG_TENSOR_TIMEOUTS,
                         ctx->alarm_dev, B, A, ldb, lda, g_wait_limit.load(std::memory_order_relaxed), g_withhold.load(std::memory_order_relaxed)};
  cudaError_t e;
  if (half)
    e = tma ? launch_weight_grad<__half, true>(ctx, a, ma, mb, dW, c, units, s) : launch_weight_grad<__half, false>(ctx, a, ma, mb, dW, c, units, s);
  else
    e = tma ? launch_weight_grad<__nv_bfloat16, true>(ctx, a, ma, mb, dW, c, units, s)
            : launch_weight_grad<__nv_bfloat16, false>(ctx, a, ma, mb, dW, c, units, s);
  HPSPMM_CUDA_TRY(ctx, e);
  return HPSPMM_OK;
}
