// Loss of rows of logits against a teacher of whose logits only a few for each row are kept, and its gradient.
//   p     = softmax over the row's entries of (teacher / tau); an entry counts when its id lies in [0, V) and its logit is
//           above -infinity
//   loss  = tau^2 * sum_j p_j (log p_j - log softmax(z / tau)[id_j])          0 for a row without entries
//   dz_v  = dloss * tau * (softmax(z / tau)_v - sum over j with id_j = v of p_j)      zeros for a row without entries
// The teacher's rows are the values of a sparse matrix whose pattern samples the dense one, as in SDDMM.
#include <algorithm>

#include "dense_types.cuh"
#include "device_utils.cuh"
#include "hpspmm_internal.h"

namespace {

using namespace hpspmm;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxEntries = 1024;   // of the teacher for one row
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// the same value in every thread; `part` holds one float for each warp
__device__ __forceinline__ float block_max(float v, float* part) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v = fmaxf(v, part[w]);
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* part) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) v += part[w];
  return v;
}

// The teacher's entries of one row: ids (-1: does not count) and exp((t - max) / tau).  Returns how many count, with the
// largest logit and the sum of the exponentials, the same in every thread.
__device__ __forceinline__ bool load_teacher(const void* ids, int wide, const float* teacher, int64_t at, int k, int V, float c,
                                             int* id, float* e, float* part, float& top, float& total) {
  float m = -INFINITY;
  int count = 0;
  for (int j = threadIdx.x; j < k; j += kThreads) {
    const float t = teacher[at + j];
    int i = load_id(ids, wide, at + j, V);
    if (t == -INFINITY) i = -1;
    id[j] = i;
    e[j] = t;
    if (i >= 0) m = fmaxf(m, t), ++count;
  }
  top = block_max(m, part);
  const bool some = __syncthreads_or(count > 0);
  float s = 0.f;
  for (int j = threadIdx.x; j < k; j += kThreads) {
    const float v = id[j] >= 0 ? exp2_fast((e[j] - top) * c) : 0.f;
    e[j] = v;
    s += v;
  }
  total = block_sum(s, part);   // (its barriers order the writes to e as well)
  return some;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
distill_forward_kernel(int V, int k, const T* __restrict__ logits, int64_t ld, const void* __restrict__ ids, int wide,
                       const float* __restrict__ teacher, float tau, float* __restrict__ loss, float2* __restrict__ stats) {
  __shared__ int id[kMaxEntries];
  __shared__ float e[kMaxEntries], part[kWarps];
  const int64_t row = blockIdx.x;
  const T* z = logits + row * ld;
  const float c = kLog2e / tau;
  float m = -INFINITY, s = 0.f;
  for (int v = threadIdx.x; v < V; v += kThreads) {
    const float x = to_float(z[v]);
    if (x > m) {
      s *= exp2_fast((m - x) * c);
      m = x;
    }
    s += exp2_fast((x - (m == -INFINITY ? 0.f : m)) * c);
  }
  const float top = block_max(m, part);
  s = block_sum(m == -INFINITY ? s : s * exp2_fast((m - top) * c), part);
  if (threadIdx.x == 0 && stats) stats[row] = make_float2(top, s);
  float t_top, t_total;
  const bool some = load_teacher(ids, wide, teacher, row * k, k, V, c, id, e, part, t_top, t_total);
  // log p - log q = (t - t_top) / tau - log t_total - (z - top) / tau + log s
  const float apart = logf(s) - logf(t_total);
  float sum = 0.f;
  for (int j = threadIdx.x; j < k; j += kThreads)
    if (id[j] >= 0 && e[j] != 0.f)
      sum += e[j] * (((teacher[row * k + j] - t_top) - (to_float(z[id[j]]) - top)) / tau + apart);
  sum = block_sum(sum, part);
  if (threadIdx.x == 0) loss[row] = some ? sum / t_total * tau * tau : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
distill_backward_kernel(int V, int k, const T* __restrict__ logits, int64_t ld, const void* __restrict__ ids, int wide,
                        const float* __restrict__ teacher, float tau, const float2* __restrict__ stats,
                        const float* __restrict__ dloss, int64_t dloss_stride, T* __restrict__ dlogits) {
  __shared__ int id[kMaxEntries];
  __shared__ float e[kMaxEntries], part[kWarps];
  const int64_t row = blockIdx.x;
  const T* z = logits + row * ld;
  T* dz = dlogits + row * V;
  const float c = kLog2e / tau;
  float t_top, t_total;
  const bool some = load_teacher(ids, wide, teacher, row * k, k, V, c, id, e, part, t_top, t_total);
  if (!some) {
    for (int v = threadIdx.x; v < V; v += kThreads) dz[v] = from_float<T>(0.f);
    return;
  }
  const float2 st = stats[row];
  const float g = dloss[row * dloss_stride] * tau, q = 1.f / st.y;
  for (int v = threadIdx.x; v < V; v += kThreads)
    dz[v] = from_float<T>(g * (exp2_fast((to_float(z[v]) - st.x) * c) * q));
  __syncthreads();
  // the columns that the teacher names once more, each by the first of its entries
  const float per = 1.f / t_total;
  for (int j = threadIdx.x; j < k; j += kThreads) {
    const int v = id[j];
    if (v < 0) continue;
    float p = 0.f;
    bool first = true;
    for (int i = 0; i < k; ++i)
      if (id[i] == v) {
        first = first && i >= j;
        p += e[i];
      }
    if (first) dz[v] = from_float<T>(g * (exp2_fast((to_float(z[v]) - st.x) * c) * q - p * per));
  }
}

int check_distill(hpspmm_ctx* ctx, int64_t T, int64_t V, int64_t k, int32_t type, int64_t ld, int32_t id_bytes, float tau) {
  HPSPMM_REQUIRE(ctx, ctx != nullptr, "null context");
  HPSPMM_REQUIRE(ctx, T >= 0 && V >= 0 && k >= 0, "negative size");
  HPSPMM_REQUIRE(ctx, hpspmm::dense_type_size(type) != 0, "unknown element type");
  HPSPMM_REQUIRE(ctx, id_bytes == 4 || id_bytes == 8, "ids must have 4 or 8 bytes");
  HPSPMM_REQUIRE(ctx, ld >= 0, "negative row stride");
  HPSPMM_REQUIRE(ctx, tau >= 1.17549435e-38f && tau <= 3.402823466e38f, "the temperature must be positive, normal and finite");
  if (T > 2147483646ll || V > 2147483646ll) return hpspmm_unsupported(ctx, "more than 2^31 - 2 rows or columns");
  if (k > kMaxEntries) return hpspmm_unsupported(ctx, "more than 1024 entries of the teacher for a row");
  return HPSPMM_OK;
}

}  // namespace

extern "C" {

int hpspmm_topk_distill_forward(hpspmm_ctx* ctx, int64_t T, int64_t V, int64_t k, int32_t type, const void* logits,
                                int64_t ld_logits, const void* ids, int32_t id_bytes, const float* teacher_logits,
                                float temperature, float* loss, float* stats, hpspmm_stream stream) {
  HPSPMM_TRACE("hpspmm_topk_distill_forward");
  const int st = check_distill(ctx, T, V, k, type, ld_logits, id_bytes, temperature);
  if (st != HPSPMM_OK) return st;
  if (T == 0) return HPSPMM_OK;
  HPSPMM_REQUIRE(ctx, loss && (V == 0 || logits) && (k == 0 || (ids && teacher_logits)), "null pointer");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  const int wide = id_bytes == 8;
  if (type == HPSPMM_TYPE_F32)
    distill_forward_kernel<<<(unsigned)T, kThreads, 0, s>>>((int)V, (int)k, (const float*)logits, ld_logits, ids, wide,
                                                            teacher_logits, temperature, loss, (float2*)stats);
  else if (type == HPSPMM_TYPE_F16)
    distill_forward_kernel<<<(unsigned)T, kThreads, 0, s>>>((int)V, (int)k, (const __half*)logits, ld_logits, ids, wide,
                                                            teacher_logits, temperature, loss, (float2*)stats);
  else
    distill_forward_kernel<<<(unsigned)T, kThreads, 0, s>>>((int)V, (int)k, (const __nv_bfloat16*)logits, ld_logits, ids, wide,
                                                            teacher_logits, temperature, loss, (float2*)stats);
  ctx->launches++;
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

int hpspmm_topk_distill_backward(hpspmm_ctx* ctx, int64_t T, int64_t V, int64_t k, int32_t type, const void* logits,
                                 int64_t ld_logits, const void* ids, int32_t id_bytes, const float* teacher_logits,
                                 float temperature, const float* stats, const float* dloss, int64_t dloss_stride,
                                 void* dlogits, hpspmm_stream stream) {
  HPSPMM_TRACE("hpspmm_topk_distill_backward");
  const int st = check_distill(ctx, T, V, k, type, ld_logits, id_bytes, temperature);
  if (st != HPSPMM_OK) return st;
  HPSPMM_REQUIRE(ctx, dloss_stride >= 0, "negative stride");
  if (T == 0 || V == 0) return HPSPMM_OK;
  HPSPMM_REQUIRE(ctx, logits && stats && dloss && dlogits && (k == 0 || (ids && teacher_logits)), "null pointer");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  const int wide = id_bytes == 8;
  if (type == HPSPMM_TYPE_F32)
    distill_backward_kernel<<<(unsigned)T, kThreads, 0, s>>>((int)V, (int)k, (const float*)logits, ld_logits, ids, wide,
                                                             teacher_logits, temperature, (const float2*)stats, dloss,
                                                             dloss_stride, (float*)dlogits);
  else if (type == HPSPMM_TYPE_F16)
    distill_backward_kernel<<<(unsigned)T, kThreads, 0, s>>>((int)V, (int)k, (const __half*)logits, ld_logits, ids, wide,
                                                             teacher_logits, temperature, (const float2*)stats, dloss,
                                                             dloss_stride, (__half*)dlogits);
  else
    distill_backward_kernel<<<(unsigned)T, kThreads, 0, s>>>((int)V, (int)k, (const __nv_bfloat16*)logits, ld_logits, ids, wide,
                                                             teacher_logits, temperature, (const float2*)stats, dloss,
                                                             dloss_stride, (__nv_bfloat16*)dlogits);
  ctx->launches++;
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

}  // extern "C"
