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

// Rows [r0, r0 + rows) of one group: g < G a group, g >= G rows that belong to none.
struct row_tile {
  int g, r0, rows;
};

// The t-th tile of up to BM rows; called by one whole warp.  rows = 0: there is none.
template <int BM>
__device__ __forceinline__ row_tile find_row_tile(const int* offsets, int G, int R, int t) {
  const int lane = threadIdx.x & 31;
  row_tile out = {0, 0, 0};
  for (int base = 0; base < G + 2; base += 32) {
    int begin, end;
    part_bounds(offsets, G, R, base + lane, begin, end);
    const int n = max(end - begin, 0), tiles = (n + BM - 1) / BM;
    int sum = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    const unsigned past = __ballot_sync(0xffffffffu, sum > t);
    if (past) {
      const int l = __ffs(past) - 1;
      const int first = __shfl_sync(0xffffffffu, sum - tiles, l);
      const int b = __shfl_sync(0xffffffffu, begin, l), e = __shfl_sync(0xffffffffu, end, l);
      out.g = base + l;
      out.r0 = b + (t - first) * BM;
      out.rows = min(BM, e - out.r0);
      return out;
    }
    t -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return out;
}

// One tile of 64 x 64 outputs: C[i][j] = sum over k of A(i, k) * B(k, j), all of them in 32 bits.
// AK / BK: the operand's elements lie next to each other along k (otherwise along i / j).
template <typename T, bool AK, bool BK>
__device__ __forceinline__ void tile_product(const T* A, int64_t sa, const T* B, int64_t sb, int rows, int cols, int depth,
                                             T* C, int64_t sc, float (*As)[68], float (*Bs)[68]) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < depth; k0 += 16) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int e = threadIdx.x + u * kThreads;
      const int i = AK ? e >> 4 : e & 63, k = AK ? e & 15 : e >> 6;
      As[k][i] = i < rows && k0 + k < depth ? to_float(A[AK ? (int64_t)i * sa + k0 + k : (int64_t)(k0 + k) * sa + i]) : 0.f;
      const int j = BK ? e >> 4 : e & 63, kb = BK ? e & 15 : e >> 6;
      Bs[kb][j] = j < cols && k0 + kb < depth ? to_float(B[BK ? (int64_t)j * sb + k0 + kb : (int64_t)(k0 + kb) * sb + j]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) a[x] = As[k][ty * 4 + x], b[x] = Bs[k][tx * 4 + x];
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = fmaf(a[x], b[y], acc[x][y]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (ty * 4 + x < rows && tx * 4 + y < cols) C[(int64_t)(ty * 4 + x) * sc + tx * 4 + y] = from_float<T>(acc[x][y]);
}

template <typename T, bool OUT_FIRST>
__global__ void __launch_bounds__(kThreads)
grouped_product_kernel(int R, int G, int K, int N, const T* __restrict__ X, int64_t ldx, const T* __restrict__ W,
                       const int* __restrict__ offsets, T* __restrict__ Y, int col_tiles) {
  __shared__ float As[16][68], Bs[16][68];
  __shared__ row_tile shared_tile;
  const int t = blockIdx.x / col_tiles, j0 = (blockIdx.x - t * col_tiles) * 64;
  if (threadIdx.x < 32) {
    const row_tile found = find_row_tile<64>(offsets, G, R, t);
    if (threadIdx.x == 0) shared_tile = found;
  }
  __syncthreads();
  const row_tile w = shared_tile;
  if (w.rows == 0) return;
  const bool none = w.g >= G;
  const T* wg = none ? W : W + (int64_t)w.g * K * N;
  tile_product<T, true, OUT_FIRST>(X + (int64_t)w.r0 * ldx, ldx, OUT_FIRST ? wg + (int64_t)j0 * K : wg + j0,
                                   OUT_FIRST ? K : N, w.rows, min(64, N - j0), none ? 0 : K, Y + (int64_t)w.r0 * N + j0, N,
                                   As, Bs);
}

// dW[g][i][j] = sum over the rows of the group of A[r][i] * B[r][j]
template <typename T>
__global__ void __launch_bounds__(kThreads)
grouped_weight_grad_kernel(int R, int G, int I, int J, const T* __restrict__ A, int64_t lda, const T* __restrict__ B,
                           int64_t ldb, const int* __restrict__ offsets, T* __restrict__ dW, int i_tiles, int j_tiles) {
  __shared__ float As[16][68], Bs[16][68];
  int t = blockIdx.x;
  const int j0 = t % j_tiles * 64;
  t /= j_tiles;
  const int i0 = t % i_tiles * 64, g = t / i_tiles;
  int begin, end;
  part_bounds(offsets, G, R, g, begin, end);
  tile_product<T, false, false>(A + (int64_t)begin * lda + i0, lda, B + (int64_t)begin * ldb + j0, ldb, min(64, I - i0),
                                min(64, J - j0), max(end - begin, 0), dW + ((int64_t)g * I + i0) * J + j0, J, As, Bs);
}

int check_grouped(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t K, int64_t N, int32_t type) {
  HPSPMM_REQUIRE(ctx, ctx != nullptr, "null context");
  HPSPMM_REQUIRE(ctx, R >= 0 && G >= 0 && K >= 0 && N >= 0, "negative size");
  HPSPMM_REQUIRE(ctx, hpspmm::dense_type_size(type) != 0, "unknown element type");
  if (R > 2147483646ll || G > 1048576 || K > 2147483646ll || N > 2147483646ll)
    return hpspmm_unsupported(ctx, "more than 2^31 - 2 rows or columns, or 2^20 groups");
  return HPSPMM_OK;
}

template <typename T>
void launch_product(int64_t R, int64_t G, int64_t K, int64_t N, const void* X, int64_t ldx, const void* W, bool out_first,
                    const int32_t* offsets, void* Y, unsigned blocks, int col_tiles, cudaStream_t s) {
  if (out_first)
    grouped_product_kernel<T, true><<<blocks, kThreads, 0, s>>>((int)R, (int)G, (int)K, (int)N, (const T*)X, ldx, (const T*)W,
                                                                offsets, (T*)Y, col_tiles);
  else
    grouped_product_kernel<T, false><<<blocks, kThreads, 0, s>>>((int)R, (int)G, (int)K, (int)N, (const T*)X, ldx, (const T*)W,
                                                                 offsets, (T*)Y, col_tiles);
}

template <typename T>
void launch_weight_grad(int64_t R, int64_t G, int64_t I, int64_t J, const void* A, int64_t lda, const void* B, int64_t ldb,
                        const int32_t* offsets, void* dW, unsigned blocks, int i_tiles, int j_tiles, cudaStream_t s) {
  grouped_weight_grad_kernel<T><<<blocks, kThreads, 0, s>>>((int)R, (int)G, (int)I, (int)J, (const T*)A, lda, (const T*)B, ldb,
                                                            offsets, (T*)dW, i_tiles, j_tiles);
}

}  // namespace

extern "C" {

int hpspmm_grouped_product(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t K, int64_t N, int32_t type, const void* X,
                           int64_t ldx, const void* W, int32_t w_out_first, const int32_t* offsets, void* Y,
                           hpspmm_stream stream) {
  HPSPMM_TRACE("hpspmm_grouped_product");
  const int st = check_grouped(ctx, R, G, K, N, type);
  if (st != HPSPMM_OK) return st;
  HPSPMM_REQUIRE(ctx, ldx >= 0, "negative row stride");
  if (R == 0 || N == 0) return HPSPMM_OK;
  HPSPMM_REQUIRE(ctx, offsets && Y && (K == 0 || (X && (W || G == 0))), "null pointer");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  const int done = hpspmm_grouped_product_tensor(ctx, R, G, K, N, type, X, ldx, W, w_out_first != 0, offsets, Y, s);
  if (done != 1) return done;
  const int64_t col_tiles = (N + 63) / 64, blocks = ((R + 63) / 64 + G + 2) * col_tiles;
  if (blocks > 2147483647ll) return hpspmm_unsupported(ctx, "more than 2^31 - 1 tiles of 64 x 64");
  if (type == HPSPMM_TYPE_F32)
    launch_product<float>(R, G, K, N, X, ldx, W, w_out_first != 0, offsets, Y, (unsigned)blocks, (int)col_tiles, s);
  else if (type == HPSPMM_TYPE_F16)
    launch_product<__half>(R, G, K, N, X, ldx, W, w_out_first != 0, offsets, Y, (unsigned)blocks, (int)col_tiles, s);
  else
    launch_product<__nv_bfloat16>(R, G, K, N, X, ldx, W, w_out_first != 0, offsets, Y, (unsigned)blocks, (int)col_tiles, s);
  ctx->launches++;
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

int hpspmm_grouped_weight_grad(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t K, int64_t N, int32_t type, const void* X,
                               int64_t ldx, const void* dY, int64_t ldy, const int32_t* offsets, void* dW,
                               int32_t w_out_first, hpspmm_stream stream) {
  HPSPMM_TRACE("hpspmm_grouped_weight_grad");
  const int st = check_grouped(ctx, R, G, K, N, type);
  if (st != HPSPMM_OK) return st;
  HPSPMM_REQUIRE(ctx, ldx >= 0 && ldy >= 0, "negative row stride");
  if (G == 0 || K == 0 || N == 0) return HPSPMM_OK;
  HPSPMM_REQUIRE(ctx, offsets && dW && (R == 0 || (X && dY)), "null pointer");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  // the operand whose columns are the rows of dW comes first
  const int64_t I = w_out_first ? N : K, J = w_out_first ? K : N;
  const void *A = w_out_first ? dY : X, *B = w_out_first ? X : dY;
  const int64_t lda = w_out_first ? ldy : ldx, ldb = w_out_first ? ldx : ldy;
  const int done = hpspmm_grouped_weight_grad_tensor(ctx, R, G, I, J, type, A, lda, B, ldb, offsets, dW, s);
  if (done != 1) return done;
  const int64_t i_tiles = (I + 63) / 64, j_tiles = (J + 63) / 64;
  if (i_tiles * j_tiles > 2147483647ll / G) return hpspmm_unsupported(ctx, "more than 2^31 - 1 tiles of 64 x 64");
  const unsigned blocks = (unsigned)(G * i_tiles * j_tiles);
  if (type == HPSPMM_TYPE_F32)
    launch_weight_grad<float>(R, G, I, J, A, lda, B, ldb, offsets, dW, blocks, (int)i_tiles, (int)j_tiles, s);
  else if (type == HPSPMM_TYPE_F16)
    launch_weight_grad<__half>(R, G, I, J, A, lda, B, ldb, offsets, dW, blocks, (int)i_tiles, (int)j_tiles, s);
  else
    launch_weight_grad<__nv_bfloat16>(R, G, I, J, A, lda, B, ldb, offsets, dW, blocks, (int)i_tiles, (int)j_tiles, s);
  ctx->launches++;
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

}  // extern "C"
