// Groups of rows: what the kernels of the grouped products share.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "device_utils.cuh"
#include "hpspmm_internal.h"

namespace hpspmm {

// Bounds of part i of the rows: the groups, then the rows behind the last and in front of the first one.  Offsets are
// taken into [0, R], so that whatever they hold no row outside the operands is named.
__device__ __forceinline__ void part_bounds(const int* offsets, int G, int R, int i, int& begin, int& end) {
  begin = end = 0;
  if (i < G) {
    begin = min(max(ld_chained(offsets + i), 0), R);
    end = min(max(ld_chained(offsets + i + 1), 0), R);
  } else if (i == G) {
    begin = min(max(ld_chained(offsets + G), 0), R);
    end = R;
  } else if (i == G + 1) {
    end = min(max(ld_chained(offsets), 0), R);
  }
}

// How the gradient of the matrices is shared out: the rows of a group in pieces of up to `length`, at least one piece for
// every group.  A group of one piece writes its matrix, the pieces of the others go to slots of 32-bit matrices that are
// added up behind.  slots: how many of them there are (for offsets that ascend no more are needed).
struct piece_plan {
  int length, slots;
};
constexpr int64_t kMostRows = 2147483647 - 1025;   // and columns: what the kernels add to fill a last tile stays below 2^31
constexpr int64_t kMostDepth = 1 << 27;   // of one tile on the tensor cores: 0.6 s with TMA, 2 to 4.4 s without
constexpr int kMostSplitGroups = 2048;   // calls of more groups are not split: they have tiles enough
__host__ __device__ __forceinline__ int pieces_of(int rows, int length) { return rows > length ? (rows - 1) / length + 1 : 1; }

// Room for the pieces of all groups that have more than one: fewer than 2 R / length.
static inline int64_t piece_slots(int64_t R, int64_t length) { return length >= R ? 0 : 2 * R / length + 1; }

}  // namespace hpspmm

// dW[g] = sum of the slots of group g, for the groups with more than one piece.
int hpspmm_join_pieces(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t elements, int32_t type, const int32_t* offsets,
                       const hpspmm::piece_plan& p, const float* slots, void* dW, cudaStream_t s);

// The tensor-core kernels, for 16-bit types.
int hpspmm_grouped_product_tensor(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t K, int64_t N, int32_t type, const void* X, int64_t ldx,
                                  const void* W, bool out_first, const int32_t* offsets, void* Y, cudaStream_t s);
int hpspmm_grouped_weight_grad_tensor(hpspmm_ctx* ctx, int64_t R, int64_t G, int64_t I, int64_t J, int32_t type, const void* A,
                                      int64_t lda, const void* B, int64_t ldb, const int32_t* offsets, void* dW,
                                      const hpspmm::piece_plan& p, float* slots, cudaStream_t s);
