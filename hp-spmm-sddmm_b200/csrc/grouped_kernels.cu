// Products of groups of rows with one matrix each, and the gradient of the matrices.
//   Y[r]  = X[r] * W[g]       for offsets[g] <= r < offsets[g + 1];  rows of no group become zeros
//   dW[g] = X_g^T * dY_g      over the rows of group g;  a group without rows gets zeros
// (dX is the first one again, with dY and the matrices the other way round.)
#include <algorithm>

#include "dense_types.cuh"
#include "device_utils.cuh"
#include "grouped.cuh"
#include "hpspmm_internal.h"

namespace {

using namespace hpspmm;

constexpr int kThreads = 256;

// ---- which rows a block has ------------------------------------------------------------------------------------------

struct row_tile {
  int g, r0, rows;   // rows [r0, r0 + rows) of part g (grouped.cuh); rows = 0: there is none
  int pieces, slot;  // gradients: pieces of the group, and where this one's goes
};

// The t-th tile of up to `length` rows, of the parts (products) or of the groups (gradients: at least one for each).  Called
// by one whole warp, which looks at 128 of them at a time.
template <bool GRADIENT>
__device__ __forceinline__ row_tile find_row_tile(const int* offsets, int G, int R, int length, int t) {
  const int lane = threadIdx.x & 31, parts = GRADIENT ? G : G + 2;
  row_tile out = {0, 0, 0, 0, 0};
  int slots_before = 0;
  for (int base = 0; base < parts; base += 128) {
    int begin[4], end[4], tiles[4], sum = 0, slots = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) part_bounds(offsets, G, R, base + lane * 4 + i, begin[i], end[i]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = max(end[i] - begin[i], 0);
      if (GRADIENT)
        tiles[i] = base + lane * 4 + i < G ? pieces_of(n, length) : 0;
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
            out.g = base + lane * 4 + i;
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
// A tile of 128 x BN outputs to a block of 256 threads, 8 x BN / 16 of them to a thread, in 32 bits from the operands on;
// 16 of the depth at a time through two buffers of shared memory, the next ones on their way to registers meanwhile.
// Bound by the multiply-adds, two of which go as one packed instruction (fma.rn.f32x2).

constexpr int kTileRows = 128;
constexpr int kTileDepth = 16;

__device__ __forceinline__ void fma_pair(uint64_t& acc, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}
__device__ __forceinline__ uint64_t both(float v) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(v));
  return r;
}

// ROWS x 16 elements of an operand; element (i, k) lies at p[i * stride + k] (ALONG: next to each other along the depth) or
// p[k * stride + i].  VEC: four neighbours are one aligned load, or none of them is there.
template <int ROWS, bool ALONG, bool VEC>
struct tile_loader {
  static constexpr int kEach = ROWS * kTileDepth / kThreads / 4;   // quads to a thread
  float v[kEach][4];
  __device__ __forceinline__ void load(const float* p, int64_t stride, int rows, int depth, int k0) {
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int q = threadIdx.x + u * kThreads;
      const int i = ALONG ? q >> 2 : q % (ROWS / 4) * 4, k = k0 + (ALONG ? (q & 3) * 4 : q / (ROWS / 4));
      const float* at = p + (ALONG ? i * stride + k : k * stride + i);
      const bool line = ALONG ? i < rows : k < depth;
      const int left = !line ? 0 : (ALONG ? depth - k : rows - i);
      if (VEC) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (left > 0) x = __ldg(reinterpret_cast<const float4*>(at));
        v[u][0] = x.x, v[u][1] = x.y, v[u][2] = x.z, v[u][3] = x.w;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[u][e] = e < left ? __ldg(at + e) : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(float (*s)[ROWS + 4]) const {
#pragma unroll
    for (int u = 0; u < kEach; ++u) {
      const int q = threadIdx.x + u * kThreads;
      if (ALONG) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[(q & 3) * 4 + e][q >> 2] = v[u][e];
      } else {
        *reinterpret_cast<float4*>(&s[q / (ROWS / 4)][q % (ROWS / 4) * 4]) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
      }
    }
  }
};

// C[i][j] = sum over k < depth of A(i, k) * B(k, j) for i < rows, j < cols.
template <int BN, bool A_ALONG, bool B_ALONG, bool VEC>
__device__ __forceinline__ void tile_product(const float* A, int64_t sa, const float* B, int64_t sb, int rows, int cols, int depth, float* C,
                                             int64_t sc, float (*As)[kTileDepth][kTileRows + 4], float (*Bs)[kTileDepth][BN + 4]) {
  constexpr int kHalves = BN / 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  uint64_t acc[8][kHalves * 2];
#pragma unroll
  for (int x = 0; x < 8; ++x)
#pragma unroll
    for (int y = 0; y < kHalves * 2; ++y) acc[x][y] = 0;
  tile_loader<kTileRows, A_ALONG, VEC> la;
  tile_loader<BN, B_ALONG, VEC> lb;
  la.load(A, sa, rows, depth, 0), lb.load(B, sb, cols, depth, 0);
  la.store(As[0]), lb.store(Bs[0]);
  __syncthreads();
  int buf = 0;
  for (int k0 = 0; k0 < depth; k0 += kTileDepth) {
    const bool more = k0 + kTileDepth < depth;
    if (more) la.load(A, sa, rows, depth, k0 + kTileDepth), lb.load(B, sb, cols, depth, k0 + kTileDepth);
#pragma unroll
    for (int k = 0; k < kTileDepth; ++k) {
      float a[8];
      uint64_t b[kHalves * 2];
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<float4*>(a + 4 * h) = *reinterpret_cast<const float4*>(&As[buf][k][ty * 4 + 64 * h]);
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
        *reinterpret_cast<ulonglong2*>(b + 2 * h) = *reinterpret_cast<const ulonglong2*>(&Bs[buf][k][tx * 4 + 64 * h]);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const uint64_t aa = both(a[x]);
#pragma unroll
        for (int y = 0; y < kHalves * 2; ++y) fma_pair(acc[x][y], aa, b[y]);
      }
    }
    if (more) {
      la.store(As[buf ^ 1]), lb.store(Bs[buf ^ 1]);
      __syncthreads();
      buf ^= 1;
    }
  }
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const int i = ty * 4 + (x & 3) + (x >> 2) * 64;
    if (i >= rows) continue;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int j = tx * 4 + 64 * h;
      float* to = C + (int64_t)i * sc + j;
      float v[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        v[2 * e] = __uint_as_float((uint32_t)acc[x][2 * h + e]);
        v[2 * e + 1] = __uint_as_float((uint32_t)(acc[x][2 * h + e] >> 32));
      }
      if (VEC) {
        if (j < cols) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < cols) to[e] = v[e];
      }
    }
  }
}

template <int BN, bool OUT_FIRST, bool VEC>
__global__ void __launch_bounds__(kThreads, 2)
grouped_product_kernel(int R, int G, int K, int N, const float* __restrict__ X, int64_t ldx, const float* __restrict__ W, const int* offsets,
                       float* __restrict__ Y, int col_tiles) {
  __shared__ float As[2][kTileDepth][kTileRows + 4], Bs[2][kTileDepth][BN + 4];
  __shared__ row_tile shared_tile;
  const int t = blockIdx.x / col_tiles, j0 = (blockIdx.x - t * col_tiles) * BN;
  if (threadIdx.x < 32) {
    const row_tile found = find_row_tile<false>(offsets, G, R, kTileRows, t);
    if (threadIdx.x == 0) shared_tile = found;
  }
  __syncthreads();
  const row_tile w = shared_tile;
  if (w.rows == 0) return;
  const bool none = w.g >= G;
  const float* wg = none ? W : W + (int64_t)w.g * K * N;
  tile_product<BN, true, OUT_FIRST, VEC>(X + (int64_t)w.r0 * ldx, ldx, OUT_FIRST ? wg + (int64_t)j0 * K : wg + j0, OUT_FIRST ? K : N,
                                               w.rows, min(BN, N - j0), none ? 0 : K, Y + (int64_t)w.r0 * N + j0, N, As, Bs);
}

// dW[g][i][j] = sum over the rows of the group of A[r][i] * B[r][j]
template <int BN, bool VEC>
__global__ void __launch_bounds__(kThreads, 2)
grouped_weight_grad_kernel(int R, int G, int I, int J, const float* __restrict__ A, int64_t lda, const float* __restrict__ B, int64_t ldb,
                           const int* offsets, float* __restrict__ dW, const piece_plan plan, float* slots, int i_tiles, int j_tiles) {
  __shared__ float As[2][kTileDepth][kTileRows + 4], Bs[2][kTileDepth][BN + 4];
  __shared__ row_tile shared_tile;
  int t = blockIdx.x;
  const int j0 = t % j_tiles * BN;
  t /= j_tiles;
  const int i0 = t % i_tiles * kTileRows;
  t /= i_tiles;
  if (threadIdx.x < 32) {
    const row_tile found = find_row_tile<true>(offsets, G, R, plan.length, t);
    if (threadIdx.x == 0) shared_tile = found;
  }
  __syncthreads();
  const row_tile w = shared_tile;
  if (w.pieces == 0 || (w.pieces > 1 && w.slot >= plan.slots)) return;
  const float *a = A + (int64_t)w.r0 * lda + i0, *b = B + (int64_t)w.r0 * ldb + j0;
  const int rows = min(kTileRows, I - i0), cols = min(BN, J - j0);
  float* to = w.pieces == 1 ? dW + (int64_t)w.g * I * J : slots + (int64_t)w.slot * I * J;
  tile_product<BN, false, false, VEC>(a, lda, b, ldb, rows, cols, w.rows, to + (int64_t)i0 * J + j0, J, As, Bs);
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

template <int BN, bool OUT_FIRST, bool VEC>
void launch_product(int64_t R, int64_t G, int64_t K, int64_t N, const void* X, int64_t ldx, const void* W, const int32_t* offsets,
                    void* Y, cudaStream_t s) {
  const int64_t col_tiles = (N + BN - 1) / BN, blocks = ((R + kTileRows - 1) / kTileRows + G + 2) * col_tiles;
  grouped_product_kernel<BN, OUT_FIRST, VEC><<<(unsigned)blocks, kThreads, 0, s>>>((int)R, (int)G, (int)K, (int)N, (const float*)X, ldx,
                                                                                  (const float*)W, offsets, (float*)Y, (int)col_tiles);
}

template <int BN, bool VEC>
void launch_weight_grad(int64_t R, int64_t G, int64_t I, int64_t J, const void* A, int64_t lda, const void* B, int64_t ldb,
                        const int32_t* offsets, void* dW, const piece_plan& p, float* slots, cudaStream_t s) {
  const int64_t i_tiles = (I + kTileRows - 1) / kTileRows, j_tiles = (J + BN - 1) / BN;
  const int64_t blocks = (G + piece_slots(R, p.length)) * i_tiles * j_tiles;
  grouped_weight_grad_kernel<BN, VEC><<<(unsigned)blocks, kThreads, 0, s>>>((int)R, (int)G, (int)I, (int)J, (const float*)A, lda,
                                                                           (const float*)B, ldb, offsets, (float*)dW, p, slots, (int)i_tiles,
                                                                              (int)j_tiles);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Columns of a tile: 64 where that covers the output, as a matrix of a relation type often is that narrow.
int64_t tile_columns(int64_t cols) { return cols <= 64 ? 64 : 128; }

// Rows to a piece.  Ordinary cores: enough pieces for four blocks on each SM, if they have 256 rows (a tile takes about 10 us
// for them); tensor cores: for two rounds of the SMs, if they have 1024 rows (about 4 us, against 2 to 3 for the 128 KB of a
// tile in 32 bits).  All the rows where there are tiles enough.
piece_plan plan_pieces(int64_t R, int64_t G, int64_t I, int64_t J, int32_t type) {
  const bool f32 = type == HPSPMM_TYPE_F32;
  const int64_t bi = f32 ? kTileRows : 256, bj = f32 ? tile_columns(J) : 128;
  const int64_t tiles = ((I + bi - 1) / bi) * ((J + bj - 1) / bj), target = 148 * (f32 ? 4 : 2);
  int64_t length = R;
  if (tiles < target && G <= kMostSplitGroups) length = std::max<int64_t>(f32 ? 256 : 1024, (R * tiles / target + 63) / 64 * 64);
  length = std::max<int64_t>(1, std::min(length, R));
  return {(int)length, (int)piece_slots(R, length)};
}

int check_grouped(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t K, int64_t N, int32_t type) {
  HPSPMM_REQUIRE(ctx, R >= 0 && G >= 0 && K >= 0 && N >= 0, "negative size");
  HPSPMM_REQUIRE(ctx, hpspmm::dense_type_size(type) != 0, "unknown element type");
  if (R > 2147483646ll || G > 1048576 || K > 2147483646ll || N > 2147483646ll)
    return hpspmm_unsupported(ctx, "more than 2^31 - 2 rows or columns, or 2^20 groups");
  return HPSPMM_OK;
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

template <int BN, bool VEC>
void launch_product(bool out_first, int64_t R, int64_t G, int64_t K, int64_t N, const void* X, int64_t ldx, const void* W,
                    const int32_t* offsets, void* Y, cudaStream_t s) {
  if (out_first)
    launch_product<BN, true, VEC>(R, G, K, N, X, ldx, W, offsets, Y, s);
  else
    launch_product<BN, false, VEC>(R, G, K, N, X, ldx, W, offsets, Y, s);
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
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  if (K == 0 || G == 0) {
    HPSPMM_CUDA_TRY(ctx, cudaMemsetAsync(Y, 0, (size_t)(R * N) * dense_type_size(type), s));
    return HPSPMM_OK;
  }
  if (type != HPSPMM_TYPE_F32)
    return hpspmm_grouped_product_tensor(ctx, R, G, K, N, type, X, ldx, W, w_out_first != 0, offsets, Y, s);
  if (((R + kTileRows - 1) / kTileRows + G + 2) * ((N + 63) / 64) > 2147483647ll)
    return hpspmm_unsupported(ctx, "more than 2^31 - 1 tiles of 128 x 64");
  const bool vec = K % 4 == 0 && N % 4 == 0 && ldx % 4 == 0 && aligned16(X) && aligned16(W) && aligned16(Y);
  const bool narrow = tile_columns(N) == 64, of = w_out_first != 0;
  if (vec && narrow)
    launch_product<64, true>(of, R, G, K, N, X, ldx, W, offsets, Y, s);
  else if (vec)
    launch_product<128, true>(of, R, G, K, N, X, ldx, W, offsets, Y, s);
  else if (narrow)
    launch_product<64, false>(of, R, G, K, N, X, ldx, W, offsets, Y, s);
  else
    launch_product<128, false>(of, R, G, K, N, X, ldx, W, offsets, Y, s);
  ctx->launches++;
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
    const int done = hpspmm_grouped_weight_grad_tensor(ctx, R, G, I, J, type, A, lda, B, ldb, offsets, dW, p, slots, s);
    if (done != HPSPMM_OK) return done;
  } else {
    if ((G + p.slots) * ((I + kTileRows - 1) / kTileRows) * ((J + 63) / 64) > 2147483647ll)
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
