// Helpers of the operators on rows of channels (embedding, gated scan, experts): the three floating types, 32-bit arithmetic
// on them, and pieces of a row as one access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

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

// The same as 32-bit words in registers: V * sizeof(T) is 2 (in the low half) or a multiple of 4.
template <class T, int V> struct words {
  static constexpr int BYTES = (int)sizeof(T) * V, N = BYTES < 4 ? 1 : BYTES / 4;
  unsigned at[N];
};
template <class T, int V> __device__ __forceinline__ words<T, V> load_words(const T* p) {
  words<T, V> w;
  if constexpr (words<T, V>::BYTES == 2) w.at[0] = *reinterpret_cast<const unsigned short*>(p);
  else if constexpr (words<T, V>::BYTES == 4) w.at[0] = *reinterpret_cast<const unsigned*>(p);
  else if constexpr (words<T, V>::BYTES == 8) { const uint2 u = *reinterpret_cast<const uint2*>(p); w.at[0] = u.x; w.at[1] = u.y; }
  else { const uint4 u = *reinterpret_cast<const uint4*>(p); w.at[0] = u.x; w.at[1] = u.y; w.at[2] = u.z; w.at[3] = u.w; }
  return w;
}
template <class T, int V> __device__ __forceinline__ void store_words(T* p, const words<T, V>& w) {
  if constexpr (words<T, V>::BYTES == 2) *reinterpret_cast<unsigned short*>(p) = (unsigned short)w.at[0];
  else if constexpr (words<T, V>::BYTES == 4) *reinterpret_cast<unsigned*>(p) = w.at[0];
  else if constexpr (words<T, V>::BYTES == 8) *reinterpret_cast<uint2*>(p) = make_uint2(w.at[0], w.at[1]);
  else *reinterpret_cast<uint4*>(p) = make_uint4(w.at[0], w.at[1], w.at[2], w.at[3]);
}
// channel v of them as a float; all of them from floats
template <int v, class T, int V> __device__ __forceinline__ float channel(const words<T, V>& w) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w.at[v]);
  else if constexpr (std::is_same<T, bf16>::value) return __uint_as_float(v % 2 ? w.at[v / 2] & 0xffff0000u : w.at[v / 2] << 16);
  else return __half2float(__ushort_as_half((unsigned short)(v % 2 ? w.at[v / 2] >> 16 : w.at[v / 2])));
}
template <class T, int V> __device__ __forceinline__ words<T, V> to_words(const float (&f)[V]) {
  words<T, V> w;
#pragma unroll
  for (int i = 0; i < words<T, V>::N; ++i) {
    if constexpr (sizeof(T) == 4) w.at[i] = __float_as_uint(f[i]);
    else if constexpr (V == 1) w.at[i] = std::is_same<T, bf16>::value ? (unsigned)__bfloat16_as_ushort(__float2bfloat16_rn(f[0])) : (unsigned)__half_as_ushort(__float2half_rn(f[0]));
    else if constexpr (std::is_same<T, bf16>::value) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w.at[i] = *reinterpret_cast<const unsigned*>(&b);
    } else {
      const __half2 b = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w.at[i] = *reinterpret_cast<const unsigned*>(&b);
    }
  }
  return w;
}
template <int N, class F> __device__ __forceinline__ void each(F f) {
  if constexpr (N > 0) { each<N - 1>(f); f(std::integral_constant<int, N - 1>()); }
}
template <class T, int V> __device__ __forceinline__ void channels(const words<T, V>& w, float (&f)[V]) {
  each<V>([&](auto v) { f[decltype(v)::value] = channel<decltype(v)::value>(w); });
}

// how many threads take a row's pieces side by side, as a power of two: enough to cover them, up to 2^most
inline unsigned spread_of(size_t pieces, unsigned most) {
  unsigned g = 0;
  while (g < most && (size_t(1) << g) < pieces) ++g;
  return g;
}
// which of the groups of 2^spread threads this thread is in is `part` of `parts` of item `at`
struct share { size_t at; unsigned part, in; };
__device__ __forceinline__ share share_of(size_t thread, unsigned spread, unsigned parts) {
  const size_t group = thread >> spread;
  share s;
  s.at = parts == 1 ? group : group <= 0xffffffffull ? (size_t)((unsigned)group / parts) : group / parts;
  s.part = (unsigned)(group - s.at * parts);
  s.in = (unsigned)thread & ((1u << spread) - 1);
  return s;
}

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
