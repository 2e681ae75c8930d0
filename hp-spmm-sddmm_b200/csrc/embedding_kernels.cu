// Rows of a table by id, and the gradient of the table.
//   out[t]    = scale * table[id[t]]                       a row of zeros where id[t] lies outside [0, N)
//   dTable[v] = scale * sum over t with id[t] = v of dOut[t]
// It is the product of a pattern with one entry to a row, and the product of its transpose, without a CSR of either.
#include <algorithm>

#include "dense_types.cuh"
#include "device_utils.cuh"
#include "hpspmm_internal.h"

namespace {

using namespace hpspmm;

constexpr int kThreads = 256;

// One thread to a vector of the output.
template <typename T, int BYTES>
__global__ void __launch_bounds__(kThreads)
lookup_kernel(int64_t total, int per_row, int N, const void* __restrict__ ids, int wide, const T* __restrict__ table,
              int64_t ld, float scale, T* __restrict__ out) {
  typedef dense_vec<T, BYTES> vec;
  const int64_t stride = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += stride) {
    const int64_t t = i / per_row;
    const int c = (int)(i - t * per_row) * vec::kCount;
    const int id = load_id(ids, wide, t, N);
    vec v;
    if (id >= 0) {
      v.raw = *reinterpret_cast<const decltype(v.raw)*>(table + (int64_t)id * ld + c);
#pragma unroll
      for (int e = 0; e < vec::kCount; ++e) v.at[e] = from_float<T>(scale * to_float(v.at[e]));
    } else {
#pragma unroll
      for (int e = 0; e < vec::kCount; ++e) v.at[e] = from_float<T>(0.f);
    }
    reinterpret_cast<decltype(v.raw)*>(out)[i] = v.raw;
  }
}

// Place of every position in the order of (id, position): how many come before it.  Ids outside the table count as N.
__global__ void __launch_bounds__(kThreads)
rank_kernel(int T, int N, const void* __restrict__ ids, int wide, int* __restrict__ key_out, int* __restrict__ pos_out) {
  __shared__ int keys[kThreads];
  const int t = blockIdx.x * kThreads + threadIdx.x;
  int mine = N;
  if (t < T) {
    const int id = load_id(ids, wide, t, N);
    if (id >= 0) mine = id;
  }
  int rank = 0;
  for (int base = 0; base < T; base += kThreads) {
    __syncthreads();
    int k = 0x7fffffff;
    if (base + (int)threadIdx.x < T) {
      const int id = load_id(ids, wide, base + threadIdx.x, N);
      k = id >= 0 ? id : N;
    }
    keys[threadIdx.x] = k;
    __syncthreads();
    const int n = min(kThreads, T - base);
    for (int j = 0; j < n; ++j) rank += keys[j] < mine || (keys[j] == mine && base + j < t);
  }
  if (t < T) {
    key_out[rank] = mine;
    pos_out[rank] = t;
  }
}

// One warp to a row of the table: the sorted positions of its id, in ascending order.
template <typename T>
__global__ void __launch_bounds__(kThreads)
sum_rows_kernel(int T_, int N, int K, const int* __restrict__ keys, const int* __restrict__ pos, const T* __restrict__ dout,
                int64_t ld, float scale, T* __restrict__ dtable) {
  const int lane = threadIdx.x & 31;
  for (int64_t v = ((int64_t)blockIdx.x * kThreads + threadIdx.x) >> 5; v < N; v += ((int64_t)gridDim.x * kThreads) >> 5) {
    int lo = 0, hi = T_;
    while (lo < hi) {
      const int m = lo + (hi - lo) / 2;
      if (keys[m] < v) lo = m + 1; else hi = m;
    }
    for (int c = lane; c < K; c += 32) {
      float sum = 0.f;
      for (int j = lo; j < T_ && keys[j] == v; ++j) sum += to_float(dout[pos[j] * ld + c]);
      dtable[v * K + c] = from_float<T>(scale * sum);
    }
  }
}

template <typename T, int BYTES>
void launch_lookup(hpspmm_ctx* ctx, int64_t T_, int64_t N, int64_t K, const void* ids, int wide, const void* table,
                   int64_t ld, float scale, void* out, cudaStream_t s) {
  const int per_row = (int)(K * (int64_t)sizeof(T) / BYTES);
  const int64_t total = T_ * per_row;
  const int64_t blocks = std::min<int64_t>((total + kThreads - 1) / kThreads, (int64_t)ctx->sm_count * 32);
  lookup_kernel<T, BYTES><<<(unsigned)blocks, kThreads, 0, s>>>(total, per_row, (int)N, ids, wide, (const T*)table, ld,
                                                                scale, (T*)out);
}

template <typename T>
void launch_lookup_of(hpspmm_ctx* ctx, int64_t T_, int64_t N, int64_t K, const void* ids, int wide, const void* table,
                      int64_t ld, float scale, void* out, cudaStream_t s) {
  const int bytes = dense_vector_bytes((uintptr_t)table | (uintptr_t)out | (uintptr_t)(K * (int64_t)sizeof(T)) |
                                           (uintptr_t)(ld * (int64_t)sizeof(T)), (int)sizeof(T));
  if (bytes == 16)
    launch_lookup<T, 16>(ctx, T_, N, K, ids, wide, table, ld, scale, out, s);
  else if (bytes == 8)
    launch_lookup<T, 8>(ctx, T_, N, K, ids, wide, table, ld, scale, out, s);
  else if (bytes == 4 || sizeof(T) == 4)
    launch_lookup<T, 4>(ctx, T_, N, K, ids, wide, table, ld, scale, out, s);
  else
    launch_lookup<T, sizeof(T)>(ctx, T_, N, K, ids, wide, table, ld, scale, out, s);
}

int check_embedding(hpspmm_ctx* ctx, int64_t T, int64_t N, int64_t K, int32_t type, int32_t id_bytes, int64_t ld) {
  HPSPMM_REQUIRE(ctx, ctx != nullptr, "null context");
  HPSPMM_REQUIRE(ctx, T >= 0 && N >= 0 && K >= 0, "negative size");
  HPSPMM_REQUIRE(ctx, hpspmm::dense_type_size(type) != 0, "unknown element type");
  HPSPMM_REQUIRE(ctx, id_bytes == 4 || id_bytes == 8, "ids must have 4 or 8 bytes");
  HPSPMM_REQUIRE(ctx, ld >= 0, "negative row stride");
  if (T > 2147483646ll || N > 2147483646ll || K > 2147483646ll)
    return hpspmm_unsupported(ctx, "more than 2^31 - 2 positions, rows or columns");
  return HPSPMM_OK;
}

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

}  // namespace

extern "C" {

int hpspmm_embedding_forward(hpspmm_ctx* ctx, int64_t T, int64_t N, int64_t K, int32_t type, const void* ids,
                             int32_t id_bytes, const void* table, int64_t ld_table, float scale, void* out,
                             hpspmm_stream stream) {
  HPSPMM_TRACE("hpspmm_embedding_forward");
  const int st = check_embedding(ctx, T, N, K, type, id_bytes, ld_table);
  if (st != HPSPMM_OK) return st;
  HPSPMM_REQUIRE(ctx, ld_table >= K, "row stride below the number of columns");
  if (T == 0 || K == 0) return HPSPMM_OK;
  HPSPMM_REQUIRE(ctx, ids && out && (table || N == 0), "null pointer");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  if (type == HPSPMM_TYPE_F32)
    launch_lookup_of<float>(ctx, T, N, K, ids, id_bytes == 8, table, ld_table, scale, out, s);
  else if (type == HPSPMM_TYPE_F16)
    launch_lookup_of<__half>(ctx, T, N, K, ids, id_bytes == 8, table, ld_table, scale, out, s);
  else
    launch_lookup_of<__nv_bfloat16>(ctx, T, N, K, ids, id_bytes == 8, table, ld_table, scale, out, s);
  ctx->launches++;
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

int64_t hpspmm_embedding_backward_workspace(int64_t T, int64_t N, int64_t K) {
  if (T < 0 || N < 0 || K < 0 || T > 2147483646ll || N > 2147483646ll || K > 2147483646ll) return -1;
  return (int64_t)(2 * align_up((size_t)T * 4, 256));
}

int hpspmm_embedding_backward(hpspmm_ctx* ctx, int64_t T, int64_t N, int64_t K, int32_t type, const void* ids,
                              int32_t id_bytes, const void* dOut, int64_t ld_dout, float scale, void* dTable,
                              void* workspace, size_t workspace_bytes, hpspmm_stream stream) {
  HPSPMM_TRACE("hpspmm_embedding_backward");
  const int st = check_embedding(ctx, T, N, K, type, id_bytes, ld_dout);
  if (st != HPSPMM_OK) return st;
  if (N == 0 || K == 0) return HPSPMM_OK;
  HPSPMM_REQUIRE(ctx, dTable && (T == 0 || (ids && dOut && workspace)), "null pointer");
  HPSPMM_REQUIRE(ctx, (int64_t)workspace_bytes >= hpspmm_embedding_backward_workspace(T, N, K), "workspace too small");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  int* keys = (int*)workspace;
  int* pos = (int*)((char*)workspace + align_up((size_t)T * 4, 256));
  if (T > 0) {
    rank_kernel<<<(unsigned)((T + kThreads - 1) / kThreads), kThreads, 0, s>>>((int)T, (int)N, ids, id_bytes == 8, keys, pos);
    ctx->launches++;
    HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  }
  const unsigned blocks = (unsigned)std::min<int64_t>((N + 7) / 8, (int64_t)ctx->sm_count * 64);
  if (type == HPSPMM_TYPE_F32)
    sum_rows_kernel<<<blocks, kThreads, 0, s>>>((int)T, (int)N, (int)K, keys, pos, (const float*)dOut, ld_dout, scale, (float*)dTable);
  else if (type == HPSPMM_TYPE_F16)
    sum_rows_kernel<<<blocks, kThreads, 0, s>>>((int)T, (int)N, (int)K, keys, pos, (const __half*)dOut, ld_dout, scale, (__half*)dTable);
  else
    sum_rows_kernel<<<blocks, kThreads, 0, s>>>((int)T, (int)N, (int)K, keys, pos, (const __nv_bfloat16*)dOut, ld_dout, scale,
                                                (__nv_bfloat16*)dTable);
  ctx->launches++;
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

}  // extern "C"
