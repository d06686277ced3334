// C ABI: tb200_expert_dispatch, tb200_expert_combine and tb200_expert_combine_grad.
#include "abi_rows.cuh"

using namespace tb200_abi;
using namespace tb200_rows;

namespace {
constexpr int BLOCK = 128;
constexpr int MOST_EXPERTS = 1024;
constexpr int MOST_CHOICES = 32;

// Stable counting sort of m ids by one CTA: counts, their prefixes, then 1024 ids at a time in order.
template <class I>
__global__ void __launch_bounds__(1024) expert_places_kernel(const I* ids, unsigned m, unsigned experts, int* slots, int* sources, int* offsets) {
  __shared__ unsigned next[MOST_EXPERTS];
  __shared__ unsigned id_at[1024];
  const unsigned t = threadIdx.x;
  next[t] = 0;
  __syncthreads();
  for (unsigned i = t; i < m; i += 1024) {
    const long long e = (long long)ids[i];
    if (e >= 0 && e < (long long)experts) atomicAdd(&next[(unsigned)e], 1u);
  }
  __syncthreads();
  if (t == 0) {
    unsigned sum = 0;
    for (unsigned e = 0; e < experts; ++e) { const unsigned c = next[e]; next[e] = sum; offsets[e] = (int)sum; sum += c; }
    offsets[experts] = (int)sum;
  }
  __syncthreads();
  for (unsigned base = 0; base < m; base += 1024) {
    const unsigned i = base + t;
    const long long e = i < m ? (long long)ids[i] : -1;
    const bool kept = e >= 0 && e < (long long)experts;
    id_at[t] = kept ? (unsigned)e : ~0u;
    __syncthreads();
    unsigned before = 0, all = 0;
    if (kept)
      for (unsigned j = 0; j < 1024; ++j) { const bool same = id_at[j] == (unsigned)e; all += same; before += same && j < t; }
    unsigned at = 0;
    if (kept) at = next[(unsigned)e] + before;
    __syncthreads();
    if (kept) { slots[i] = (int)at; sources[at] = (int)i; if (before == 0) next[(unsigned)e] += all; }
    else if (i < m) slots[i] = -1;
    __syncthreads();
  }
  for (unsigned i = (unsigned)offsets[experts] + t; i < m; i += 1024) sources[i] = -1;
}

// a CTA a row
template <class T>
__global__ void __launch_bounds__(BLOCK) expert_rows_kernel(const T* x, size_t xs, const int* sources, unsigned choices, size_t dim, T* rows) {
  const int source = sources[blockIdx.x];
  T* const to = rows + (size_t)blockIdx.x * dim;
  for (size_t c = threadIdx.x; c < dim; c += BLOCK) to[c] = source < 0 ? from_f32<T>(0.f) : x[(size_t)((unsigned)source / choices) * xs + c];
}

// out[token] = sum of weights * rows over the token's choices that have a place; a CTA a token
template <class T>
__global__ void __launch_bounds__(BLOCK) expert_combine_kernel(const T* rows, size_t rs, size_t m, const int* slots, const float* weights, unsigned choices, size_t dim, T* out) {
  const size_t token = blockIdx.x;
  for (size_t c = threadIdx.x; c < dim; c += BLOCK) {
    float sum = 0.f;
    for (unsigned k = 0; k < choices; ++k) {
      const int at = slots[token * choices + k];
      if ((unsigned)at < m) sum += (weights ? weights[token * choices + k] : 1.f) * to_f32(rows[(size_t)at * rs + c]);
    }
    out[token * dim + c] = from_f32<T>(sum);
  }
}

// drows[place] = weight * dout[token], dweight = <dout[token], rows[place]>; a CTA a token, and one more for each row without a source
template <class T>
__global__ void __launch_bounds__(BLOCK) expert_combine_grad_kernel(const T* dout, size_t ds, const T* rows, size_t rs, size_t m, const int* slots, const float* weights,
                                                                  const int* end, size_t n, unsigned choices, size_t dim, T* drows, float* dweights) {
  __shared__ float part[BLOCK / 32];
  if (blockIdx.x >= n) {
    const size_t row = blockIdx.x - n;
    if ((long long)row < (long long)*end) return;
    for (size_t c = threadIdx.x; c < dim; c += BLOCK) drows[row * dim + c] = from_f32<T>(0.f);
    return;
  }
  const size_t token = blockIdx.x;
  for (unsigned k = 0; k < choices; ++k) {
    const int at = slots[token * choices + k];
    const bool kept = (unsigned)at < m;
    const float w = kept ? weights[token * choices + k] : 0.f;
    float dot = 0.f;
    if (kept)
      for (size_t c = threadIdx.x; c < dim; c += BLOCK) {
        const float d = to_f32(dout[token * ds + c]);
        dot += d * to_f32(rows[(size_t)at * rs + c]);
        drows[(size_t)at * dim + c] = from_f32<T>(w * d);
      }
    for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(tb200::FULL_MASK, dot, o);
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = dot;
    __syncthreads();
    if (threadIdx.x == 0) dweights[token * choices + k] = (part[0] + part[1]) + (part[2] + part[3]);
    __syncthreads();
  }
}

// what every one of these calls needs of its sizes: flat assignments and rows are counted in 31 bits
bool sizes_fit(size_t n, size_t choices) { return choices >= 1 && choices <= (size_t)MOST_CHOICES && n <= 0x7fffffffull / choices / 2; }
}  // namespace

TB200_API int tb200_expert_dispatch(const void* d_x, size_t x_stride, const void* d_experts, int expert_t, size_t n, size_t choices, size_t num_experts, size_t dim, int t,
                                    void* d_rows, int* d_slots, int* d_sources, int* d_offsets, void* d_ws, size_t* ws_bytes, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    return by_index_dtype(expert_t, [&](auto iv) -> int {
      using I = decltype(iv);
      if (!sizes_fit(n, choices) || num_experts < 1 || num_experts > (size_t)MOST_EXPERTS) return ERR_INVALID;
      int rc;
      if (workspace_gate(d_ws, ws_bytes, sizeof(tb200::ws_header), rc)) return rc;
      const unsigned m = (unsigned)(n * choices);
      if (!d_offsets || (m && (!d_experts || !d_slots || !d_sources || (dim && (!d_x || !d_rows)))) || x_stride < dim) return ERR_INVALID;
      expert_places_kernel<I><<<1, 1024, 0, stream>>>(static_cast<const I*>(d_experts), m, (unsigned)num_experts, d_slots, d_sources, d_offsets);
      if (m && dim) expert_rows_kernel<T><<<m, BLOCK, 0, stream>>>(static_cast<const T*>(d_x), x_stride, d_sources, (unsigned)choices, dim, static_cast<T*>(d_rows));
      return (int)cudaGetLastError();
    });
  });
}

TB200_API int tb200_expert_combine(const void* d_rows, size_t rows_stride, const int* d_slots, const float* d_weights, size_t n, size_t choices, size_t dim, int t, void* d_out,
                                   tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    if (!sizes_fit(n, choices)) return ERR_INVALID;
    if (n == 0 || dim == 0) return 0;
    if (!d_rows || !d_slots || !d_out || rows_stride < dim) return ERR_INVALID;
    expert_combine_kernel<T><<<(unsigned)n, BLOCK, 0, stream>>>(static_cast<const T*>(d_rows), rows_stride, n * choices, d_slots, d_weights, (unsigned)choices, dim, static_cast<T*>(d_out));
    return (int)cudaGetLastError();
  });
}

TB200_API int tb200_expert_combine_grad(const void* d_dout, size_t dout_stride, const void* d_rows, size_t rows_stride, const int* d_slots, const float* d_weights,
                                        const int* d_kept, size_t n, size_t choices, size_t dim, int t, void* d_drows, float* d_dweights, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    if (!sizes_fit(n, choices)) return ERR_INVALID;
    if (n == 0) return 0;
    if (!d_slots || !d_weights || !d_kept || !d_dweights || (dim && (!d_dout || !d_rows || !d_drows)) || dout_stride < dim || rows_stride < dim) return ERR_INVALID;
    const size_t m = n * choices;
    expert_combine_grad_kernel<T><<<(unsigned)(n + m), BLOCK, 0, stream>>>(static_cast<const T*>(d_dout), dout_stride, static_cast<const T*>(d_rows), rows_stride, m, d_slots, d_weights,
                                                                         d_kept, n, (unsigned)choices, dim, static_cast<T*>(d_drows), d_dweights);
    return (int)cudaGetLastError();
  });
}
