// Products of groups of rows with one matrix each, and the gradient of the matrices.
//   Y[r]  = X[r] * W[g]       for offsets[g] <= r < offsets[g + 1];  rows of no group become zeros
//   dW[g] = X_g^T * dY_g      over the rows of group g;  a group without rows gets zeros
// (dX is the first one again, with dY and the matrices the other way round.)
#include <algorithm>
#include <cmath>

#include "dense_types.cuh"
#include "device_utils.cuh"
#include "grouped.cuh"
#include "hpspmm_internal.h"

namespace {

using namespace hpspmm;

constexpr int kThreads = 256;

// ---- which rows a block has ------------------------------------------------------------------------------------------

// Parts that one launch of a product has.  Every block looks through them for its own, 128 at a time (so a multiple of that),
// and with all of many in one launch the time grew with their square: 131,072 groups of 1,000 rows, 16 x 16: 118 ms, now 1.5.
// 200,000 rows of 4,000 groups take 124 us in one launch and 123 in two.
constexpr int kMostSearched = 33 * 128;

struct row_tile {
  int g, r0, rows;   // rows [r0, r0 + rows) of part g (grouped.cuh); rows = 0: there is none
  int pieces, slot;  // gradients: pieces of the group, and where this one's goes
};

// The t-th tile of up to `length` rows, of the `parts` parts from g0 on (products) or of the groups (gradients: at least one
// for each).  Called by whole warps, each of which looks at 128 of them at a time; kMostSearched bounds their number.
template <bool GRADIENT>
__device__ __forceinline__ row_tile find_row_tile(const int* offsets, int G, int R, int length, int t, int g0, int parts) {
  const int lane = threadIdx.x & 31;
  row_tile out = {0, 0, 0, 0, 0};
  int slots_before = 0;
  for (int base = 0; base < parts; base += 128) {
    int begin[4], end[4], tiles[4], sum = 0, slots = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) part_bounds(offsets, G, R, g0 + base + lane * 4 + i, begin[i], end[i]);   // (none behind G + 2)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = max(end[i] - begin[i], 0);
      if (GRADIENT)
        tiles[i] = base + lane * 4 + i < parts ? pieces_of(n, length) : 0;
      else
        tiles[i] = (n + length - 1) / length;
      sum += tiles[i];
      if (tiles[i] > 1) slots += tiles[i];
    }
    sum = min(sum, 1 << 25), slots = min(slots, 1 << 25);   // (offsets that do not ascend: 32 of them stay below 2^31)
    int before = sum, before_slots = slots;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, before, d), p = __shfl_up_sync(0xffffffffu, before_slots, d);
      if (lane >= d) before += o, before_slots += p;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before > t);
    if (past) {
      const int l = __ffs(past) - 1;
      if (lane == l) {
        int left = t - (before - sum), slot = slots_before + before_slots - slots;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (left >= 0 && left < tiles[i]) {
            out.g = g0 + base + lane * 4 + i;
            out.r0 = begin[i] + left * length;
            out.rows = max(min(length, end[i] - out.r0), 0);
            out.pieces = tiles[i], out.slot = slot + left;
            left = -1;
          } else {
            left -= left >= 0 ? tiles[i] : 0;
            if (tiles[i] > 1) slot += tiles[i];
          }
        }
      }
      out.g = __shfl_sync(0xffffffffu, out.g, l), out.r0 = __shfl_sync(0xffffffffu, out.r0, l);
      out.rows = __shfl_sync(0xffffffffu, out.rows, l), out.pieces = __shfl_sync(0xffffffffu, out.pieces, l);
      out.slot = __shfl_sync(0xffffffffu, out.slot, l);
      return out;
    }
    t -= __shfl_sync(0xffffffffu, before, 31);
    slots_before += __shfl_sync(0xffffffffu, before_slots, 31);
  }
  return out;
}

// ---- products on the ordinary cores --------------------------------------------------------------------------------
//
// A tile of TR x BN outputs to a block of 2 TR threads, 8 x BN / 16 of them to a thread, in 32 bits from the operands on;
// 16 of the depth at a time, copied asynchronously into a ring of three buffers in the order in which they lie in memory.
// Bound by the multiply-adds (60 % of the pipe's cycles for 100,003 rows of 47 groups, 100 x 64), two of which go as one packed instruction (fma.rn.f32x2): on two neighbouring columns of the
// output, or, where both operands lie along the depth, on two neighbours of it, whose sums meet at the end.
// TR = 64 for products, whose depth is short as often as not, so that more blocks hide each other's beginnings (100,003 x 100
// by 47 matrices of 64: 46 us with 128, 41 with 64); 128 for gradients, which read less that way (55 us with 64, 46 with 128).

constexpr int kProductRows = 64;    // of a tile
constexpr int kGradientRows = 128;
constexpr int kTileDepth = 16;
constexpr int kBuffers = 3;

__device__ __forceinline__ void fma_pair(uint64_t& acc, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}
__device__ __forceinline__ uint64_t both(float v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float half_of(uint64_t v, int h) { return __uint_as_float((uint32_t)(v >> (32 * h))); }

// zeros where `there` is false (nothing is read then)
template <int BYTES>
__device__ __forceinline__ void copy_async(float* dst, const float* src, bool there) {
  const unsigned to = (unsigned)__cvta_generic_to_shared(dst);
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(there ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(src), "r"(there ? 4 : 0) : "memory");
}

// ROWS x 16 elements of an operand; element (i, k) lies at p[i * stride + k] (ALONG: next to each other along the depth, and
// so in the buffer: 20 floats to a row, which keeps the reads of 8 rows off each other's banks) or at p[k * stride + i].
// VEC: four neighbours are one aligned copy, or none of them is there.
template <int ROWS, int THREADS, bool ALONG, bool VEC>
struct operand_tile {
  static constexpr int kPitch = ALONG ? kTileDepth + 4 : ROWS;
  static constexpr int kFloats = (ALONG ? ROWS : kTileDepth) * kPitch;
  static __device__ __forceinline__ void copy(float* s, const float* p, int64_t stride, int rows, int depth, int k0) {
#pragma unroll
    for (int u = 0; u < ROWS * kTileDepth / THREADS / 4; ++u) {
      const int q = threadIdx.x + u * THREADS;
      const int line = ALONG ? q >> 2 : q / (ROWS / 4), in = (ALONG ? q & 3 : q % (ROWS / 4)) * 4;
      const int i = ALONG ? line : in, k = k0 + (ALONG ? in : line);
      const int left = ALONG ? (i < rows ? depth - k : 0) : (k < depth ? rows - i : 0);
      const float* at = p + (ALONG ? i * stride + k : k * stride + i);
      float* to = s + line * kPitch + in;
      if (VEC) {
        copy_async<16>(to, left > 0 ? at : p, left > 0);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) copy_async<4>(to + e, e < left ? at + e : p, e < left);
      }
    }
  }
};

template <int TR, int BN, bool A_ALONG, bool B_ALONG, bool VEC>
struct tile_shape {
  typedef operand_tile<TR, 2 * TR, A_ALONG, VEC> a;
  typedef operand_tile<BN, 2 * TR, B_ALONG, VEC> b;
  static constexpr int kBytes = kBuffers * (a::kFloats + b::kFloats) * 4;
};

// C[i][j] = sum over k < depth of A(i, k) * B(k, j) for i < rows, j < cols.
template <int TR, int BN, bool A_ALONG, bool B_ALONG, bool VEC>
__device__ __forceinline__ void tile_product(const float* A, int64_t sa, const float* B, int64_t sb, int rows, int cols, int depth, float* C,
                                             int64_t sc, float* smem) {
  typedef tile_shape<TR, BN, A_ALONG, B_ALONG, VEC> shape;
  typedef typename shape::a ta;
  typedef typename shape::b tb;
  static_assert(!B_ALONG || (A_ALONG && BN == 64), "two along the depth take twice the accumulators");
  constexpr bool kDeep = A_ALONG && B_ALONG;
  constexpr int kHalves = BN / 64, kAcc = kDeep ? 4 : 2 * kHalves;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  auto row_of = [&](int x) { return ty * 4 + (x & 3) + (x >> 2) * (TR / 2); };
  float* const bs = smem + kBuffers * ta::kFloats;
  const int steps = (depth + kTileDepth - 1) / kTileDepth;
  auto fetch = [&](int step) {
    if (step < steps) {
      ta::copy(smem + step % kBuffers * ta::kFloats, A, sa, rows, depth, step * kTileDepth);
      tb::copy(bs + step % kBuffers * tb::kFloats, B, sb, cols, depth, step * kTileDepth);
    }
    cp_async_commit();
  };
  uint64_t acc[8][kAcc];
#pragma unroll
  for (int x = 0; x < 8; ++x)
#pragma unroll
    for (int y = 0; y < kAcc; ++y) acc[x][y] = 0;
#pragma unroll
  for (int i = 0; i < kBuffers - 1; ++i) fetch(i);
  for (int step = 0; step < steps; ++step) {
    cp_async_wait<kBuffers - 2>();
    __syncthreads();
    fetch(step + kBuffers - 1);      // into the buffer that everybody has left
    const float *as = smem + step % kBuffers * ta::kFloats, *b0 = bs + step % kBuffers * tb::kFloats;
#pragma unroll
    for (int k = 0; k < kTileDepth; k += 4) {
      if (kDeep) {
        ulonglong2 a[8], b[4];
#pragma unroll
        for (int x = 0; x < 8; ++x) a[x] = *reinterpret_cast<const ulonglong2*>(as + row_of(x) * ta::kPitch + k);
#pragma unroll
        for (int y = 0; y < 4; ++y) b[y] = *reinterpret_cast<const ulonglong2*>(b0 + (tx + 16 * y) * tb::kPitch + k);
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
          for (int y = 0; y < kAcc; ++y) fma_pair(acc[x][y], a[x].x, b[y % 4].x), fma_pair(acc[x][y], a[x].y, b[y % 4].y);
      } else {
        float a[4][8];   // [k][x]
        if (A_ALONG) {
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const float4 v = *reinterpret_cast<const float4*>(as + row_of(x) * ta::kPitch + k);
            a[0][x] = v.x, a[1][x] = v.y, a[2][x] = v.z, a[3][x] = v.w;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              *reinterpret_cast<float4*>(&a[i][4 * h]) = *reinterpret_cast<const float4*>(as + (k + i) * ta::kPitch + ty * 4 + TR / 2 * h);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint64_t b[2 * kHalves];
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            *reinterpret_cast<ulonglong2*>(b + 2 * h) = *reinterpret_cast<const ulonglong2*>(b0 + (k + i) * tb::kPitch + tx * 4 + 64 * h);
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const uint64_t aa = both(a[i][x]);
#pragma unroll
            for (int y = 0; y < 2 * kHalves; ++y) fma_pair(acc[x][y % kAcc], aa, b[y]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    if (row_of(x) >= rows) continue;
    float* to = C + (int64_t)row_of(x) * sc;
    if (kDeep) {
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (tx + 16 * y < cols) to[tx + 16 * y] = half_of(acc[x][y % kAcc], 0) + half_of(acc[x][y % kAcc], 1);
    } else {
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const int j = tx * 4 + 64 * h;
        const float v[4] = {half_of(acc[x][2 * h % kAcc], 0), half_of(acc[x][2 * h % kAcc], 1), half_of(acc[x][(2 * h + 1) % kAcc], 0),
                            half_of(acc[x][(2 * h + 1) % kAcc], 1)};
        if (VEC) {
          if (j < cols) *reinterpret_cast<float4*>(to + j) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (j + e < cols) to[j + e] = v[e];
        }
      }
    }
  }
}

template <int BN, bool OUT_FIRST, bool VEC>
__global__ void __launch_bounds__(2 * kProductRows, BN == 64 && !OUT_FIRST ? 5 : 4)
grouped_product_kernel(int R, int G, int K, int N, const float* __restrict__ X, int64_t ldx, const float* __restrict__ W, const int* offsets,
                       float* __restrict__ Y, int col_tiles, int g0, int parts) {
  extern __shared__ float4 tile_smem[];
  const int t = blockIdx.x / col_tiles, j0 = (blockIdx.x - t * col_tiles) * BN;
  const row_tile w = find_row_tile<false>(offsets, G, R, kProductRows, t, g0, parts);
  if (w.rows == 0) return;
  const bool none = w.g >= G;
  const float* wg = none ? W : W + (int64_t)w.g * K * N;
  tile_product<kProductRows, BN, true, OUT_FIRST, VEC>(X + (int64_t)w.r0 * ldx, ldx, OUT_FIRST ? wg + (int64_t)j0 * K : wg + j0, OUT_FIRST ? K : N,
                                               w.rows, min(BN, N - j0), none ? 0 : K, Y + (int64_t)w.r0 * N + j0, N,
                                         reinterpret_cast<float*>(tile_smem));
}

// dW[g][i][j] = sum over the rows of the group of A[r][i] * B[r][j]
template <int BN, bool VEC>
__global__ void __launch_bounds__(2 * kGradientRows, 2)
grouped_weight_grad_kernel(int R, int G, int I, int J, const float* __restrict__ A, int64_t lda, const float* __restrict__ B, int64_t ldb,
                           const int* offsets, float* __restrict__ dW, const piece_plan plan, float* slots, int i_tiles, int j_tiles) {
  extern __shared__ float4 tile_smem[];
  int t = blockIdx.x;
  const int j0 = t % j_tiles * BN;
  t /= j_tiles;
  const int i0 = t % i_tiles * kGradientRows;
  t /= i_tiles;
  row_tile w;
  if (plan.slots > 0) {
    w = find_row_tile<true>(offsets, G, R, plan.length, t, 0, G);
  } else {   // groups as they are
    int end;
    part_bounds(offsets, G, R, t, w.r0, end);
    w.g = t, w.rows = max(end - w.r0, 0), w.pieces = 1;
  }
  if (w.pieces == 0 || (w.pieces > 1 && w.slot >= plan.slots)) return;
  const float *a = A + (int64_t)w.r0 * lda + i0, *b = B + (int64_t)w.r0 * ldb + j0;
  const int rows = min(kGradientRows, I - i0), cols = min(BN, J - j0);
  float* to = w.pieces == 1 ? dW + (int64_t)w.g * I * J : slots + (int64_t)w.slot * I * J;
  tile_product<kGradientRows, BN, false, false, VEC>(a, lda, b, ldb, rows, cols, w.rows, to + (int64_t)i0 * J + j0, J,
                                      reinterpret_cast<float*>(tile_smem));
}

// Groups of more than one piece: the pieces in order.
template <typename T>
__global__ void __launch_bounds__(kThreads)
join_pieces_kernel(int R, int G, int64_t elements, const int* offsets, const piece_plan plan, const float* slots, T* __restrict__ dW) {
  __shared__ int part[kThreads / 32];
  const int g = blockIdx.y;
  int begin, end;
  part_bounds(offsets, G, R, g, begin, end);
  const int pieces = pieces_of(max(end - begin, 0), plan.length);
  if (pieces == 1) return;
  int before = 0;
  for (int i = threadIdx.x; i < g; i += kThreads) {
    part_bounds(offsets, G, R, i, begin, end);
    const int n = pieces_of(max(end - begin, 0), plan.length);
    if (n > 1) before += n;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) before += __shfl_xor_sync(0xffffffffu, before, d);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = before;
  __syncthreads();
  before = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) before += part[w];
  const int last = min(before + pieces, plan.slots);
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < elements; e += (int64_t)gridDim.x * kThreads) {
    float sum = 0.f;
#pragma unroll 8
    for (int s = before; s < last; ++s) sum += slots[s * elements + e];
    dW[g * elements + e] = from_float<T>(sum);
  }
}

// (a refused size of the shared memory shows at the launch)
template <int BN, bool OUT_FIRST, bool VEC>
void launch_product(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t K, int64_t N, const void* X, int64_t ldx, const void* W, const int32_t* offsets,
                    void* Y, cudaStream_t s) {
  constexpr int smem = tile_shape<kProductRows, BN, true, OUT_FIRST, VEC>::kBytes;
  cudaFuncSetAttribute(grouped_product_kernel<BN, OUT_FIRST, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  const int64_t col_tiles = (N + BN - 1) / BN;
  for (int64_t g0 = 0; g0 < G + 2; g0 += kMostSearched) {
    const int64_t parts = std::min<int64_t>(kMostSearched, G + 2 - g0);
    const int64_t blocks = ((R + kProductRows - 1) / kProductRows + std::min(R, parts)) * col_tiles;
    grouped_product_kernel<BN, OUT_FIRST, VEC><<<(unsigned)blocks, 2 * kProductRows, smem, s>>>(
        (int)R, (int)G, (int)K, (int)N, (const float*)X, ldx, (const float*)W, offsets, (float*)Y, (int)col_tiles, (int)g0, (int)parts);
    ctx->launches++;
  }
}

template <int BN, bool VEC>
void launch_weight_grad(int64_t R, int64_t G, int64_t I, int64_t J, const void* A, int64_t lda, const void* B, int64_t ldb,
                        const int32_t* offsets, void* dW, const piece_plan& p, float* slots, cudaStream_t s) {
  constexpr int smem = tile_shape<kGradientRows, BN, false, false, VEC>::kBytes;
  cudaFuncSetAttribute(grouped_weight_grad_kernel<BN, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  const int64_t i_tiles = (I + kGradientRows - 1) / kGradientRows, j_tiles = (J + BN - 1) / BN;
  const int64_t blocks = (G + piece_slots(R, p.length)) * i_tiles * j_tiles;
  grouped_weight_grad_kernel<BN, VEC><<<(unsigned)blocks, 2 * kGradientRows, smem, s>>>(
      (int)R, (int)G, (int)I, (int)J, (const float*)A, lda, (const float*)B, ldb, offsets, (float*)dW, p, slots, (int)i_tiles, (int)j_tiles);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Columns of a tile: 64 where that covers the output, as a matrix of a relation type often is that narrow.
int64_t tile_columns(int64_t cols) { return cols <= 64 ? 64 : 128; }

// Rows to a piece: all of them, or as many as fill the GPU once where that is expected to be faster.  In us: what 64 rows
// take a tile (0.30 to 0.47 on the tensor cores, less with fewer tiles, which are smaller then, 1.65 without TMA; 9.6 or, 64
// columns wide, 4.8 on the ordinary ones, which run two of them on an SM); whole groups take as long as the largest one,
// for which twice the mean is assumed; pieces have at least 1024 (256) rows, take another launch and the way of their sums
// to memory and back (4 TB/s; somewhat more than half of the slots are used).  16 groups of 750 rows, 1024 x 1024: 73 us in
// pieces, 31 whole; one group of 12,000, 4096 x 512: 59 us in pieces, 71 whole; in 32 bits 16 groups of 750 rows, 512 x
// 512: 175 us in pieces, 270 whole.
piece_plan plan_pieces(int64_t R, int64_t G, int64_t I, int64_t J, int32_t type) {
  const bool f32 = type == HPSPMM_TYPE_F32;
  const int64_t bi = f32 ? kGradientRows : 256, bj = f32 ? tile_columns(J) : 128, least = f32 ? 256 : 1024;
  const int64_t tiles = ((I + bi - 1) / bi) * ((J + bj - 1) / bj), at_once = f32 ? 296 : 148;
  piece_plan whole = {(int)std::max<int64_t>(1, R), 0};
  if (G > kMostSplitGroups || R <= least || tiles >= at_once) return whole;
  const int64_t length = std::min(R, std::max(least, (R * tiles / at_once + 63) / 64 * 64));
  const piece_plan p = {(int)length, (int)piece_slots(R, length)};
  const bool lines = I % 8 != 0 || J % 8 != 0;   // rows that TMA does not take
  const double us = f32 ? (bj == 64 ? 4.8 : 9.6) : (lines ? 1.65 : 0.47);
  const double us_whole = f32 || lines || G * tiles >= 100 ? us : (G * tiles < 50 ? 0.3 : 0.4);
  const double rows = (double)R, largest = G == 1 ? rows : std::min(rows, 2 * rows / (double)G);
  const double t_whole = std::ceil((double)(G * tiles) / (double)at_once) * largest / 64 * us_whole;
  const double t_pieces = rows * (double)tiles / 64 * us / (double)at_once + 0.6 * (double)length / 64 * us + 7 +
                          0.6 * (double)p.slots * (double)I * (double)J * 8 / 4e6;
  return t_pieces < t_whole ? p : whole;
}

int check_grouped(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t K, int64_t N, int32_t type) {
  HPSPMM_REQUIRE(ctx, R >= 0 && G >= 0 && K >= 0 && N >= 0, "negative size");
  HPSPMM_REQUIRE(ctx, hpspmm::dense_type_size(type) != 0, "unknown element type");
  if (R > kMostRows || G > 1048576 || K > kMostRows || N > kMostRows)
    return hpspmm_unsupported(ctx, "more than 2^31 - 1026 rows or columns, or 2^20 groups");
  return ctx ? hpspmm_report_timeout(ctx) : HPSPMM_OK;
}

}  // namespace

int hpspmm_join_pieces(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t elements, int32_t type, const int32_t* offsets,
                       const piece_plan& p, const float* slots, void* dW, cudaStream_t s) {
  const dim3 grid((unsigned)std::min<int64_t>((elements + kThreads - 1) / kThreads, std::max<int64_t>(1, 8 * ctx->sm_count / G)), (unsigned)G);
  if (type == HPSPMM_TYPE_F32)
    join_pieces_kernel<<<grid, kThreads, 0, s>>>((int)R, (int)G, elements, offsets, p, slots, (float*)dW);
  else if (type == HPSPMM_TYPE_F16)
    join_pieces_kernel<<<grid, kThreads, 0, s>>>((int)R, (int)G, elements, offsets, p, slots, (__half*)dW);
  else
    join_pieces_kernel<<<grid, kThreads, 0, s>>>((int)R, (int)G, elements, offsets, p, slots, (__nv_bfloat16*)dW);
  ctx->launches++;
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

extern "C" {

int hpspmm_grouped_product(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t K, int64_t N, int32_t type, const void* X,
                           int64_t ldx, const void* W, int32_t w_out_first, const int32_t* offsets, void* Y,
                           hpspmm_stream stream) {
  HPSPMM_TRACE("hpspmm_grouped_product");
  HPSPMM_REQUIRE(ctx, ctx != nullptr, "null context");
  const int st = check_grouped(ctx, R, G, K, N, type);
  if (st != HPSPMM_OK) return st;
  HPSPMM_REQUIRE(ctx, ldx >= 0, "negative row stride");
  if (R == 0 || N == 0) return HPSPMM_OK;
  HPSPMM_REQUIRE(ctx, offsets && Y && (K == 0 || (X && (W || G == 0))), "null pointer");
  const int size = dense_type_size(type);
  HPSPMM_REQUIRE(ctx, may_begin(offsets, 4) && may_begin(Y, size) && may_begin(X, size) && may_begin(W, size),
                 "an array does not begin on a multiple of its elements' size");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  if (K == 0 || G == 0) {
    HPSPMM_CUDA_TRY(ctx, cudaMemsetAsync(Y, 0, (size_t)(R * N) * dense_type_size(type), s));
    return HPSPMM_OK;
  }
  if (type != HPSPMM_TYPE_F32 && K > kMostDepth) return hpspmm_unsupported(ctx, "16-bit products deeper than 2^27");
  if (type != HPSPMM_TYPE_F32)
    return hpspmm_grouped_product_tensor(ctx, R, G, K, N, type, X, ldx, W, w_out_first != 0, offsets, Y, s);
  if (((R + kProductRows - 1) / kProductRows + std::min<int64_t>(G + 2, kMostSearched)) * ((N + 63) / 64) > 2147483647ll)
    return hpspmm_unsupported(ctx, "more than 2^31 - 1 tiles of 64 x 64");
  const bool vec = K % 4 == 0 && N % 4 == 0 && ldx % 4 == 0 && aligned16(X) && aligned16(W) && aligned16(Y);
  const bool narrow = tile_columns(N) == 64, of = w_out_first != 0;
  if (of && vec)
    launch_product<64, true, true>(ctx, R, G, K, N, X, ldx, W, offsets, Y, s);
  else if (of)
    launch_product<64, true, false>(ctx, R, G, K, N, X, ldx, W, offsets, Y, s);
  else if (vec && narrow)
    launch_product<64, false, true>(ctx, R, G, K, N, X, ldx, W, offsets, Y, s);
  else if (vec)
    launch_product<128, false, true>(ctx, R, G, K, N, X, ldx, W, offsets, Y, s);
  else if (narrow)
    launch_product<64, false, false>(ctx, R, G, K, N, X, ldx, W, offsets, Y, s);
  else
    launch_product<128, false, false>(ctx, R, G, K, N, X, ldx, W, offsets, Y, s);
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

int64_t hpspmm_grouped_weight_grad_workspace(int64_t R, int64_t G, int64_t K, int64_t N, int32_t type, int32_t w_out_first) {
  if (check_grouped(nullptr, R, G, K, N, type) != HPSPMM_OK) return -1;
  if (R == 0 || G == 0 || K == 0 || N == 0) return 0;
  return (int64_t)plan_pieces(R, G, w_out_first ? N : K, w_out_first ? K : N, type).slots * K * N * 4;
}

int hpspmm_grouped_weight_grad(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t K, int64_t N, int32_t type, const void* X,
                               int64_t ldx, const void* dY, int64_t ldy, const int32_t* offsets, void* dW,
                               int32_t w_out_first, void* workspace, size_t workspace_bytes, hpspmm_stream stream) {
  HPSPMM_TRACE("hpspmm_grouped_weight_grad");
  HPSPMM_REQUIRE(ctx, ctx != nullptr, "null context");
  const int st = check_grouped(ctx, R, G, K, N, type);
  if (st != HPSPMM_OK) return st;
  HPSPMM_REQUIRE(ctx, ldx >= 0 && ldy >= 0, "negative row stride");
  if (G == 0 || K == 0 || N == 0) return HPSPMM_OK;
  HPSPMM_REQUIRE(ctx, offsets && dW && (R == 0 || (X && dY)), "null pointer");
  const int size = dense_type_size(type);
  HPSPMM_REQUIRE(ctx, may_begin(offsets, 4) && may_begin(dW, size) && may_begin(X, size) && may_begin(dY, size),
                 "an array does not begin on a multiple of its elements' size");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  if (R == 0) {
    HPSPMM_CUDA_TRY(ctx, cudaMemsetAsync(dW, 0, (size_t)(G * K * N) * dense_type_size(type), s));
    return HPSPMM_OK;
  }
  // the operand whose columns are the rows of dW comes first
  const int64_t I = w_out_first ? N : K, J = w_out_first ? K : N;
  const void *A = w_out_first ? dY : X, *B = w_out_first ? X : dY;
  const int64_t lda = w_out_first ? ldy : ldx, ldb = w_out_first ? ldx : ldy;
  const piece_plan p = plan_pieces(R, G, I, J, type);
  float* slots = (float*)workspace;
  if (p.slots > 0) {
    HPSPMM_REQUIRE(ctx, workspace != nullptr && (int64_t)workspace_bytes >= (int64_t)p.slots * K * N * 4, "workspace too small");
    HPSPMM_REQUIRE(ctx, ((uintptr_t)workspace & 255) == 0, "workspace not aligned to 256 bytes");
  }
  if (type != HPSPMM_TYPE_F32) {
    if (p.length > kMostDepth) return hpspmm_unsupported(ctx, "16-bit gradients over more than 2^27 rows that are not cut into pieces");
    const int done = hpspmm_grouped_weight_grad_tensor(ctx, R, G, I, J, type, A, lda, B, ldb, offsets, dW, p, slots, s);
    if (done != HPSPMM_OK) return done;
  } else {
    if ((G + p.slots) * ((I + kGradientRows - 1) / kGradientRows) * ((J + 63) / 64) > 2147483647ll)
      return hpspmm_unsupported(ctx, "more than 2^31 - 1 tiles of 128 x 64");
    const bool vec = I % 4 == 0 && J % 4 == 0 && lda % 4 == 0 && ldb % 4 == 0 && aligned16(A) && aligned16(B) &&
                     aligned16(dW);
    const bool narrow = tile_columns(J) == 64;
    if (vec && narrow)
      launch_weight_grad<64, true>(R, G, I, J, A, lda, B, ldb, offsets, dW, p, slots, s);
    else if (vec)
      launch_weight_grad<128, true>(R, G, I, J, A, lda, B, ldb, offsets, dW, p, slots, s);
    else if (narrow)
      launch_weight_grad<64, false>(R, G, I, J, A, lda, B, ldb, offsets, dW, p, slots, s);
    else
      launch_weight_grad<128, false>(R, G, I, J, A, lda, B, ldb, offsets, dW, p, slots, s);
    ctx->launches++;
    HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  }
  return p.slots > 0 ? hpspmm_join_pieces(ctx, R, G, K * N, type, offsets, p, slots, dW, s) : HPSPMM_OK;
}

}  // extern "C"
