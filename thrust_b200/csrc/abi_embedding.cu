// C ABI: tb200_embedding and tb200_embedding_grad.
#include "abi_rows.cuh"
#include "thrust_b200/radix_sort.cuh"

using namespace tb200_abi;
using namespace tb200_rows;

namespace {
constexpr int BLOCK = 128;

// out[i] = scale * weight[tokens[i]]; a CTA a token
template <class T, class I>
__global__ void __launch_bounds__(BLOCK) embedding_kernel(const T* weight, size_t rows, size_t stride, const I* tokens, size_t dim, float scale, T* out) {
  const long long tok = (long long)tokens[blockIdx.x];
  const bool there = tok >= 0 && (size_t)tok < rows;
  T* const to = out + (size_t)blockIdx.x * dim;
  for (size_t c = threadIdx.x; c < dim; c += BLOCK) to[c] = there ? from_f32<T>(scale * to_f32(weight[(size_t)tok * stride + c])) : from_f32<T>(0.f);
}

// keys: the token, or `rows` for one that is no row; positions 0, 1, ...
template <class I>
__global__ void __launch_bounds__(256) token_keys_kernel(const I* tokens, size_t n, unsigned rows, unsigned* keys, unsigned* positions) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long long tok = (long long)tokens[i];
  keys[i] = tok >= 0 && tok < (long long)rows ? (unsigned)tok : rows;
  positions[i] = (unsigned)i;
}

__device__ __forceinline__ size_t first_not_below(const unsigned* keys, size_t n, unsigned key) {
  size_t lo = 0, hi = n;
  while (lo < hi) { const size_t mid = (lo + hi) >> 1; if (keys[mid] < key) lo = mid + 1; else hi = mid; }
  return lo;
}

// out[row] (+)= scale * the sum of the gradients of its places, in their order; a CTA a row.  A sort whose wait ran out leaves NaNs.
template <class T, class O>
__global__ void __launch_bounds__(BLOCK) embedding_grad_kernel(const T* dout, size_t stride, const unsigned* keys, const unsigned* positions, size_t n, size_t dim,
                                                             float scale, bool accumulate, O* out, const tb200::ws_header* hdr) {
  const unsigned row = blockIdx.x;
  const size_t begin = first_not_below(keys, n, row), end = first_not_below(keys, n, row + 1);
  const bool failed = hdr->error != 0;
  if (begin == end && accumulate && !failed) return;
  for (size_t c = threadIdx.x; c < dim; c += BLOCK) {
    float sum = 0.f;
    for (size_t i = begin; i < end; ++i) sum += to_f32(dout[(size_t)positions[i] * stride + c]);
    sum *= scale;
    O* const to = out + (size_t)row * dim + c;
    if (accumulate) sum += to_f32(*to);
    *to = from_f32<O>(failed ? __int_as_float(0x7fffffff) : sum);
  }
}

// the workspace: the sort's, then keys, positions and the sort's other halves
struct grad_layout {
  size_t array, sort, need;
  explicit grad_layout(size_t n) {
    array = tb200::align_up(n * 4, 256);
    sort = tb200::align_up(tb200::radix_workspace_bytes<4, 4>(n), 256);
    need = sort + 4 * array;
  }
};
}  // namespace

TB200_API int tb200_embedding(const void* d_weight, size_t rows, size_t weight_stride, const void* d_tokens, int token_t, size_t n, size_t dim, int t, float scale,
                              void* d_out, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    return by_index_dtype(token_t, [&](auto iv) -> int {
      using I = decltype(iv);
      if (n == 0 || dim == 0) return 0;
      if (!d_tokens || !d_out || (rows && !d_weight) || weight_stride < dim || n > 0x7fffffffull) return ERR_INVALID;
      embedding_kernel<T, I><<<(unsigned)n, BLOCK, 0, stream>>>(static_cast<const T*>(d_weight), rows, weight_stride, static_cast<const I*>(d_tokens), dim, scale,
                                                              static_cast<T*>(d_out));
      return (int)cudaGetLastError();
    });
  });
}

TB200_API int tb200_embedding_grad(const void* d_dout, size_t dout_stride, const void* d_tokens, int token_t, size_t n, size_t rows, size_t dim, int t, int out_t,
                                   float scale, int accumulate, void* d_out, void* d_ws, size_t* ws_bytes, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    return by_row_dtype(out_t, [&](auto ov) -> int {
      using O = decltype(ov);
      return by_index_dtype(token_t, [&](auto iv) -> int {
        using I = decltype(iv);
        if (n >= (1ull << 31) || rows >= (1ull << 31)) return ERR_INVALID;
        const grad_layout lay(n);
        int rc;
        if (workspace_gate(d_ws, ws_bytes, lay.need, rc)) return rc;
        if (rows == 0 || dim == 0) return 0;
        if (!d_out || (n && (!d_dout || !d_tokens)) || dout_stride < dim) return ERR_INVALID;
        char* const base = static_cast<char*>(d_ws);
        unsigned* const keys = reinterpret_cast<unsigned*>(base + lay.sort);
        unsigned* const positions = reinterpret_cast<unsigned*>(base + lay.sort + 2 * lay.array);
        if (n) token_keys_kernel<I><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(static_cast<const I*>(d_tokens), n, (unsigned)rows, keys, positions);
        tb200::key_coding coding;
        coding.kind = tb200::KEY_UNSIGNED;
        coding.descending = 0;
        int bits = 8;
        while (bits < 32 && (rows >> bits)) bits += 8;      // the largest key is `rows`
        const cudaError_t e = tb200::radix_sort_async<uint32_t, uint32_t, true>(keys, keys + lay.array / 4, positions, positions + lay.array / 4, n, coding, 0, bits, d_ws, stream);
        if (e != cudaSuccess) return (int)e;
        embedding_grad_kernel<T, O><<<(unsigned)rows, BLOCK, 0, stream>>>(static_cast<const T*>(d_dout), dout_stride, keys, positions, n, dim, scale, accumulate != 0,
                                                                        static_cast<O*>(d_out), static_cast<const tb200::ws_header*>(d_ws));
        return (int)cudaGetLastError();
      });
    });
  });
}
