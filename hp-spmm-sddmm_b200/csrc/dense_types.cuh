// Element types of the dense operators (32, 16 and brain-16 bits) and loads and stores of short vectors of them.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "hpspmm.h"

namespace hpspmm {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
// one rounding to the nearest, ties to even
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// what BYTES bytes travel as
template <int BYTES>
struct raw_bytes;
template <>
struct raw_bytes<16> { typedef uint4 type; };
template <>
struct raw_bytes<8> { typedef uint2 type; };
template <>
struct raw_bytes<4> { typedef uint32_t type; };
template <>
struct raw_bytes<2> { typedef uint16_t type; };

// BYTES bytes of elements T, aligned to their size
template <typename T, int BYTES>
union dense_vec {
  static constexpr int kCount = BYTES / (int)sizeof(T);
  typename raw_bytes<BYTES>::type raw;
  T at[kCount];
  __device__ __forceinline__ dense_vec() {}
};

// Widest vector in bytes (16, 8, 4 or 2) that rows of `row_bytes` bytes at strides and addresses given keep aligned;
// all: the bitwise or of everything that has to be a multiple.
static inline int dense_vector_bytes(uintptr_t all, int size) {
  int b = 16;
  while (b > size && (all & (uintptr_t)(b - 1)) != 0) b >>= 1;
  return b;
}

static inline int dense_type_size(int32_t type) {
  return type == HPSPMM_TYPE_F32 ? 4 : (type == HPSPMM_TYPE_F16 || type == HPSPMM_TYPE_BF16 ? 2 : 0);
}

// Whether an array of elements of `size` bytes may begin there (a device would fault on one that may not).
static inline bool may_begin(const void* p, int size) { return ((uintptr_t)p & (uintptr_t)(size - 1)) == 0; }

// ids of 4 or 8 bytes; -1 where the id lies outside [0, n)
__device__ __forceinline__ int load_id(const void* ids, int wide, int64_t at, int n) {
  const int64_t id = wide ? static_cast<const long long*>(ids)[at] : (int64_t) static_cast<const int*>(ids)[at];
  return id >= 0 && id < n ? (int)id : -1;
}

}  // namespace hpspmm
