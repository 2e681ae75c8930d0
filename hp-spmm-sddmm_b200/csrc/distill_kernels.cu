// Loss of rows of logits against a teacher of whose logits only a few for each row are kept, and its gradient.
//   p     = softmax over the row's entries of (teacher / tau); an entry counts when its id lies in [0, V) and its logit is
//           above -infinity (so not when it is NaN)
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
constexpr int kMaxEntries = 1024;   // of the teacher for one row
// Entries that a row has room for in shared memory: 1024 to a block; to a warp 64, or 256 for teachers of more (20,000 rows of
// 2,048 bf16 and 64 entries: forward and gradient 94 us with room for 64, 111 for 256).
constexpr int kFewEntriesWarp = 64;
constexpr int kMaxEntriesWarp = 256;
// Vectors of 16 bytes in flight per thread.  4,096 x 131,072 bf16: backward 357 us with four, 346 with eight; forward with
// four 185 us where six blocks to an SM are asked for, 196 without (1,021 x 32,003 floats: 39 and 32).
constexpr int kForwardVectors = 4;
constexpr int kBackwardVectors = 8;
constexpr float kLog2e = 1.44269504088896340736f;

// (within 2^-22 of the value; results below 2^-126 are zero)
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct maximum {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct sum {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// Over the NT threads that share a row: the same value in all of them.  part: one float for each warp.
template <int NT, typename OP>
__device__ __forceinline__ float row_reduce(float v, OP op, float* part) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, d));
  if (NT == 32) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < NT / 32; ++w) v = op(v, part[w]);
  return v;
}
template <int NT>
__device__ __forceinline__ void row_sync() {
  if (NT == 32) __syncwarp(); else __syncthreads();
}
template <int NT>
__device__ __forceinline__ bool row_any(bool v) { return NT == 32 ? __any_sync(0xffffffffu, v) : __syncthreads_or(v); }

// of the blocks of a cluster
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// A row of V elements at any address: `head` elements in front of the first 16-byte boundary, vectors, the rest from `tail` on
// (which is counted from there: V may be so near 2^31 that a step past it would not be an int).
template <typename T>
struct row_parts {
  int head, vectors, tail;
  __device__ __forceinline__ row_parts(const T* p, int V) {
    constexpr int E = 16 / (int)sizeof(T);
    head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T));
    vectors = (V - head) / E;
    tail = head + vectors * E;
  }
};

// Largest value so far and the sum of exp((x - it) / tau) under it.
struct running {
  float top = -INFINITY, total = 0.f;
  // where nothing has been seen but -infinity, the difference would be no number
  static __device__ __forceinline__ float base(float top) { return top == -INFINITY ? 0.f : top; }
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N], float c) {
    float most = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) most = fmaxf(most, x[i]);
    if (most > top) {
      total *= exp2_fast((top - most) * c);
      top = most;
    }
    const float b = base(top);
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) part[i & 3] += exp2_fast((x[i] - b) * c);
    total += (part[0] + part[1]) + (part[2] + part[3]);
  }
  __device__ __forceinline__ void add(float x, float c) {
    const float v[1] = {x};
    add(v, c);
  }
  // seen under a larger value
  __device__ __forceinline__ float under(float most, float c) const {
    return top == -INFINITY ? total : total * exp2_fast((top - most) * c);
  }
};

// One pass over the row, everything in registers: NT threads to a row, CL blocks of a cluster to one where rows are few.
// Bound by the reads of the logits; an element costs one ex2 and about five other instructions.  4,096 x 131,072 bf16: 184 us,
// 5.8 TB/s; 1,021 x 32,003 floats: 32 us, 4.0 TB/s; 8 rows of 131,072 f16 in clusters of eight: 5.2 us.
template <typename T, int NT, int CL, int ENTRIES>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 6 : 0)
distill_forward_kernel(int64_t rows, int V, int k, const T* __restrict__ logits, int64_t ld, const void* __restrict__ ids, int wide,
                       const float* __restrict__ teacher, float tau, float* __restrict__ loss, float* __restrict__ stats) {
  typedef dense_vec<T, 16> vec;
  constexpr int E = vec::kCount, kTogether = 8 / E;   // eight values to a step
  constexpr int kRows = kThreads / NT, kEntries = ENTRIES;
  __shared__ float of_teacher[kRows][kEntries], of_student[kRows][kEntries];   // logits at the teacher's entries
  __shared__ float part[kThreads / 32];
  __shared__ float2 from_rank[CL];
  const int tid = threadIdx.x & (NT - 1), slot = NT == 32 ? threadIdx.x >> 5 : 0;
  const int rank = CL == 1 ? 0 : blockIdx.x & (CL - 1);
  const int64_t row = CL == 1 ? (int64_t)blockIdx.x * kRows + slot : blockIdx.x / CL;
  if (row >= rows) return;              // whole warps, and none of them in front of a barrier of the block
  // a block may write into another one's shared memory only once that one is known to run: each says so here, and waits for
  // the others behind its reads of the row
  if (CL > 1) cluster_arrive();
  const T* z = logits + row * ld;
  const float c = kLog2e / tau;
  if (rank == 0)
    for (int j = tid; j < k; j += NT) {   // an entry that does not count: -infinity
      const int id = load_id(ids, wide, row * k + j, V);
      const float t = teacher[row * k + j];
      of_teacher[slot][j] = id >= 0 && t > -INFINITY ? t : -INFINITY;   // (not one that is no number either)
      of_student[slot][j] = id >= 0 ? to_float(z[id]) : 0.f;
    }
  const row_parts<T> at(z, V);
  running r;
  if (rank == 0)
    for (int v = tid; v < at.head; v += NT) r.add(to_float(z[v]), c);
  if (rank == CL - 1)
    for (int v = tid; v < V - at.tail; v += NT) r.add(to_float(z[at.tail + v]), c);
  const uint4* words = reinterpret_cast<const uint4*>(z + at.head);
  const int begin = (int)((int64_t)at.vectors * rank / CL), end = (int)((int64_t)at.vectors * (rank + 1) / CL);
  int v = begin + tid;
  for (; v + (kForwardVectors - 1) * NT < end; v += kForwardVectors * NT) {
    vec x[kForwardVectors];
#pragma unroll
    for (int u = 0; u < kForwardVectors; ++u) x[u].raw = __ldg(words + v + u * NT);
#pragma unroll
    for (int u = 0; u < kForwardVectors; u += kTogether) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = to_float(x[u + e / E].at[e % E]);
      r.add(f, c);
    }
  }
  for (; v < end; v += NT) {
    vec x;
    x.raw = __ldg(words + v);
    float f[E];
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = to_float(x.at[e]);
    r.add(f, c);
  }
  float top = row_reduce<NT>(r.top, maximum(), part);
  float total = row_reduce<NT>(r.under(top, c), sum(), part);
  if (CL > 1) {   // the blocks' parts, in the order of their ranks
    cluster_wait();
    if (threadIdx.x == 0) {
      uint32_t to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"((uint32_t)__cvta_generic_to_shared(&from_rank[rank])));
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(top), "f"(total) : "memory");
    }
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < CL; ++i) most = fmaxf(most, from_rank[i].x);
    total = 0.f;
#pragma unroll
    for (int i = 0; i < CL; ++i) {
      running other;
      other.top = from_rank[i].x, other.total = from_rank[i].y;
      total += other.under(most, c);
    }
    top = most;
  }
  if (tid == 0 && stats) stats[2 * row] = top, stats[2 * row + 1] = total;   // (floats: they may begin on any 4 bytes)
  row_sync<NT>();
  float t_top = -INFINITY;
  for (int j = tid; j < k; j += NT) t_top = fmaxf(t_top, of_teacher[slot][j]);
  bool some = false;
  for (int j = tid; j < k; j += NT) some = some || of_teacher[slot][j] != -INFINITY;
  some = row_any<NT>(some);
  t_top = row_reduce<NT>(t_top, maximum(), part);
  float t_total = 0.f;
  for (int j = tid; j < k; j += NT) t_total += of_teacher[slot][j] == -INFINITY ? 0.f : exp2_fast((of_teacher[slot][j] - t_top) * c);
  t_total = row_reduce<NT>(t_total, sum(), part);
  // log p - log q = (t - t_top) / tau - log t_total - (z - top) / tau + log total
  const float apart = logf(total) - logf(t_total);
  float value = 0.f;
  for (int j = tid; j < k; j += NT) {
    const float t = of_teacher[slot][j], e = t == -INFINITY ? 0.f : exp2_fast((t - t_top) * c);
    if (e != 0.f) value += e * (((t - t_top) - (of_student[slot][j] - top)) / tau + apart);
  }
  value = row_reduce<NT>(value, sum(), part);
  if (tid == 0) loss[row] = some ? value / t_total * tau * tau : 0.f;
}

// Bound by memory: 4,096 x 131,072 bf16 346 us, 6.2 TB/s; 1,021 x 32,003 floats 44 us, 6.0 TB/s.
// One read and one write of the row; the columns that the teacher names are written again by the first of their entries.
// slices: blocks to a row where rows are few.  The last rows come first: the forward pass left them in the L2 cache.
template <typename T, int NT, int ENTRIES>
__global__ void __launch_bounds__(kThreads)
distill_backward_kernel(int64_t rows, int V, int k, const T* __restrict__ logits, int64_t ld, const void* __restrict__ ids, int wide,
                        const float* __restrict__ teacher, float tau, const float* __restrict__ stats,
                        const float* __restrict__ dloss, int64_t dloss_stride, T* __restrict__ dlogits, int slices) {
  typedef dense_vec<T, 16> vec;
  constexpr int E = vec::kCount;
  constexpr int kRows = kThreads / NT, kEntries = ENTRIES;
  __shared__ int id_of[kRows][kEntries];
  __shared__ float p_of[kRows][kEntries], part[kThreads / 32];
  const int tid = threadIdx.x & (NT - 1), slot = NT == 32 ? threadIdx.x >> 5 : 0;
  const int64_t back = NT == 32 ? (int64_t)blockIdx.x * kRows + slot : blockIdx.x / slices;
  const int slice = NT == 32 ? 0 : (int)(blockIdx.x - back * slices);
  if (back >= rows) return;             // whole warps, and none of them in front of a barrier of the block
  const int64_t row = rows - 1 - back;
  const T* z = logits + row * ld;
  T* dz = dlogits + row * V;
  int* id = id_of[slot];
  float* p = p_of[slot];
  const float c = kLog2e / tau;
  const float2 st = make_float2(stats[2 * row], stats[2 * row + 1]);
  const float g = dloss[row * dloss_stride] * tau, q = 1.f / st.y;
  float t_top = -INFINITY;
  bool some = false;
  for (int j = tid; j < k; j += NT) {
    const float t = teacher[row * k + j];
    const int i = t > -INFINITY ? load_id(ids, wide, row * k + j, V) : -1;
    id[j] = i, p[j] = t;
    if (i >= 0) some = true, t_top = fmaxf(t_top, t);
  }
  some = row_any<NT>(some);
  t_top = row_reduce<NT>(t_top, maximum(), part);
  float t_total = 0.f;
  for (int j = tid; j < k; j += NT) {
    const float e = id[j] >= 0 ? exp2_fast((p[j] - t_top) * c) : 0.f;
    p[j] = e;
    t_total += e;
  }
  const float per = 1.f / row_reduce<NT>(t_total, sum(), part);
  auto value = [&](float x) { return some ? g * (exp2_fast((x - st.x) * c) * q) : 0.f; };
  const row_parts<T> at(z, V), to(dz, V);
  const int body = at.head == to.head ? at.vectors : 0;
  const int begin = (int)((int64_t)body * slice / slices), end = (int)((int64_t)body * (slice + 1) / slices);
  if (at.head == to.head) {
    if (slice == 0)
      for (int v = tid; v < at.head; v += NT) dz[v] = from_float<T>(value(to_float(z[v])));
    if (slice == slices - 1)
      for (int v = tid; v < V - at.tail; v += NT) dz[at.tail + v] = from_float<T>(value(to_float(z[at.tail + v])));
  } else {   // rows of the two that begin differently: element by element
    for (int64_t v = (int64_t)V * slice / slices + tid; v < (int64_t)V * (slice + 1) / slices; v += NT)
      dz[v] = from_float<T>(value(to_float(z[v])));
  }
  const uint4* words = reinterpret_cast<const uint4*>(z + at.head);
  uint4* out = reinterpret_cast<uint4*>(dz + at.head);
  for (int v0 = begin + tid; v0 < end; v0 += kBackwardVectors * NT) {
    vec x[kBackwardVectors];
#pragma unroll
    for (int u = 0; u < kBackwardVectors; ++u)
      if (v0 + u * NT < end) x[u].raw = __ldg(words + v0 + u * NT);
#pragma unroll
    for (int u = 0; u < kBackwardVectors; ++u)
      if (v0 + u * NT < end) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[u].at[e] = from_float<T>(value(to_float(x[u].at[e])));
        out[v0 + u * NT] = x[u].raw;
      }
  }
  row_sync<NT>();
  if (!some) return;
  // the columns of this slice
  const int64_t lo = at.head != to.head ? (int64_t)V * slice / slices : (slice == 0 ? 0 : at.head + (int64_t)begin * E);
  const int64_t hi = at.head != to.head ? (int64_t)V * (slice + 1) / slices : (slice == slices - 1 ? V : at.head + (int64_t)end * E);
  for (int j = tid; j < k; j += NT) {
    const int v = id[j];
    if (v < lo || v >= hi || v < 0) continue;
    float share = 0.f;
    bool first = true;
    for (int i = 0; i < k; ++i)
      if (id[i] == v) {
        first = first && i >= j;
        share += p[i];
      }
    if (first) dz[v] = from_float<T>(g * (exp2_fast((to_float(z[v]) - st.x) * c) * q - share * per));
  }
}

// A warp to a row where rows are short; several blocks, each with at least 16 KB of it, to a row where the rows do not fill
// the SMs twice.  (Two or four to a row for more rows than that lost: 1,021 rows of 32,003 floats 32 us with one, 44 with
// four: what a row costs beside its reads comes with every block.)
struct distill_shape {
  bool warp;
  int parts;
};
distill_shape choose_distill(const hpspmm_ctx* ctx, int64_t T, int64_t V, int64_t k, int size) {
  distill_shape sh = {V * size <= 4096 && k <= kMaxEntriesWarp, 1};
  while (!sh.warp && sh.parts < 8 && T * sh.parts < 2 * ctx->sm_count && V * size >= (int64_t)sh.parts * 32768)
    sh.parts *= 2;
  return sh;
}

template <typename T, int CL>
cudaError_t launch_cluster(int64_t rows, int V, int k, const void* logits, int64_t ld, const void* ids, int wide, const float* teacher,
                           float tau, float* loss, float* stats, cudaStream_t s) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CL, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3((unsigned)(rows * CL)), c.blockDim = dim3(kThreads), c.stream = s, c.attrs = &attr, c.numAttrs = CL > 1;
  return cudaLaunchKernelEx(&c, distill_forward_kernel<T, kThreads, CL, kMaxEntries>, rows, V, k, (const T*)logits, ld, ids, wide, teacher, tau, loss,
                            stats);
}

template <typename T>
cudaError_t launch_forward(hpspmm_ctx* ctx, int64_t rows, int V, int k, const void* logits, int64_t ld, const void* ids, int wide,
                           const float* teacher, float tau, float* loss, float* stats, cudaStream_t s) {
  const distill_shape sh = choose_distill(ctx, rows, V, k, (int)sizeof(T));
  if (sh.warp) {
    auto* kernel = k <= kFewEntriesWarp ? distill_forward_kernel<T, 32, 1, kFewEntriesWarp> : distill_forward_kernel<T, 32, 1, kMaxEntriesWarp>;
    kernel<<<(unsigned)((rows + 7) / 8), kThreads, 0, s>>>(rows, V, k, (const T*)logits, ld, ids, wide, teacher, tau, loss, stats);
    return cudaSuccess;
  }
  if (sh.parts == 8) return launch_cluster<T, 8>(rows, V, k, logits, ld, ids, wide, teacher, tau, loss, stats, s);
  if (sh.parts == 4) return launch_cluster<T, 4>(rows, V, k, logits, ld, ids, wide, teacher, tau, loss, stats, s);
  if (sh.parts == 2) return launch_cluster<T, 2>(rows, V, k, logits, ld, ids, wide, teacher, tau, loss, stats, s);
  return launch_cluster<T, 1>(rows, V, k, logits, ld, ids, wide, teacher, tau, loss, stats, s);
}

template <typename T>
void launch_backward(hpspmm_ctx* ctx, int64_t rows, int V, int k, const void* logits, int64_t ld, const void* ids, int wide,
                     const float* teacher, float tau, const float* stats, const float* dloss, int64_t stride, void* dlogits,
                     cudaStream_t s) {
  const distill_shape sh = choose_distill(ctx, rows, V, k, (int)sizeof(T));
  auto* kernel = !sh.warp ? distill_backward_kernel<T, kThreads, kMaxEntries>
                 : k <= kFewEntriesWarp ? distill_backward_kernel<T, 32, kFewEntriesWarp>
                                        : distill_backward_kernel<T, 32, kMaxEntriesWarp>;
  const int64_t blocks = sh.warp ? (rows + 7) / 8 : rows * sh.parts;
  kernel<<<(unsigned)blocks, kThreads, 0, s>>>(rows, V, k, (const T*)logits, ld, ids, wide, teacher, tau, stats, dloss, stride,
                                               (T*)dlogits, sh.parts);
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
  return hpspmm_report_timeout(ctx);
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
  HPSPMM_REQUIRE(ctx, may_begin(logits, dense_type_size(type)) && may_begin(loss, 4) && may_begin(stats, 4) &&
                          (k == 0 || (may_begin(ids, id_bytes) && may_begin(teacher_logits, 4))),
                 "an array does not begin on a multiple of its elements' size");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  const int wide = id_bytes == 8;
  cudaError_t e;
  if (type == HPSPMM_TYPE_F32)
    e = launch_forward<float>(ctx, T, (int)V, (int)k, logits, ld_logits, ids, wide, teacher_logits, temperature, loss, stats, s);
  else if (type == HPSPMM_TYPE_F16)
    e = launch_forward<__half>(ctx, T, (int)V, (int)k, logits, ld_logits, ids, wide, teacher_logits, temperature, loss, stats, s);
  else
    e = launch_forward<__nv_bfloat16>(ctx, T, (int)V, (int)k, logits, ld_logits, ids, wide, teacher_logits, temperature, loss, stats, s);
  HPSPMM_CUDA_TRY(ctx, e);
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
  HPSPMM_REQUIRE(ctx, may_begin(logits, dense_type_size(type)) && may_begin(dlogits, dense_type_size(type)) && may_begin(stats, 4) &&
                          may_begin(dloss, 4) && (k == 0 || (may_begin(ids, id_bytes) && may_begin(teacher_logits, 4))),
                 "an array does not begin on a multiple of its elements' size");
  hpspmm_device_guard guard(ctx->device);
  cudaStream_t s = (cudaStream_t)stream;
  const int wide = id_bytes == 8;
  if (type == HPSPMM_TYPE_F32)
    launch_backward<float>(ctx, T, (int)V, (int)k, logits, ld_logits, ids, wide, teacher_logits, temperature, stats, dloss, dloss_stride,
                           dlogits, s);
  else if (type == HPSPMM_TYPE_F16)
    launch_backward<__half>(ctx, T, (int)V, (int)k, logits, ld_logits, ids, wide, teacher_logits, temperature, stats, dloss, dloss_stride,
                            dlogits, s);
  else
    launch_backward<__nv_bfloat16>(ctx, T, (int)V, (int)k, logits, ld_logits, ids, wide, teacher_logits, temperature, stats, dloss,
                                   dloss_stride, dlogits, s);
  ctx->launches++;
  HPSPMM_CUDA_TRY(ctx, cudaGetLastError());
  return HPSPMM_OK;
}

}  // extern "C"
