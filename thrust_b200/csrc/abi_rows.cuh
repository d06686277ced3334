// Helpers of the operators on rows of channels (embedding, gated scan, experts): the three floating types, 32-bit arithmetic
// on them, and pieces of a row as one access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "abi_common.cuh"

namespace tb200_rows {

using bf16 = __nv_bfloat16;
using f16 = __half;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(f16 x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(bf16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ f16 from_f32<f16>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float x) { return __float2bfloat16_rn(x); }

// V neighbouring channels of a row, moved in one access.
template <class T, int V> struct alignas(sizeof(T) * V) piece { T at[V]; };

// f(T()) for the type that a TB200_F32, TB200_F16 or TB200_BF16 names
template <class F> int by_row_dtype(int t, F f) {
  switch (t) {
    case TB200_F32: return f(float());
    case TB200_F16: return f(f16());
    case TB200_BF16: return f(bf16());
  }
  return tb200_abi::ERR_UNSUPPORTED;
}
template <class F> int by_index_dtype(int t, F f) {
  switch (t) {
    case TB200_I32: return f((int)0);
    case TB200_I64: return f((long long)0);
  }
  return tb200_abi::ERR_UNSUPPORTED;
}

// Whether rows of `dim` elements of `bytes` bytes, `stride` elements apart from `p` on, are made of whole aligned 16-byte pieces.
inline bool in_16_bytes(const void* p, size_t dim, size_t stride, size_t bytes) {
  return p == nullptr || ((reinterpret_cast<uintptr_t>(p) | dim * bytes | stride * bytes) & 15) == 0;
}

}  // namespace tb200_rows
