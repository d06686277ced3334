// C ABI: tb200_embedding and tb200_embedding_grad.
#include "abi_rows.cuh"
#include "thrust_b200/radix_sort.cuh"

using namespace tb200_abi;
using namespace tb200_rows;

namespace {
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

// out[i] = scale * weight[tokens[i]].  2^spread lanes take up to LOOKUP_U pieces each of a row (`parts` times that make a row): as many random reads
// are in flight per thread.  Bound by the bytes of the rows.
constexpr int LOOKUP_U = 4;
template <class T, int V, class I>
__global__ void __launch_bounds__(256) embedding_kernel(const T* __restrict__ weight, size_t rows, size_t stride, const I* __restrict__ tokens, size_t n, unsigned pieces, unsigned parts,
                                                        unsigned spread, float scale, T* __restrict__ out) {
  const share s = share_of((size_t)blockIdx.x * 256 + threadIdx.x, spread, parts);
  const size_t i = s.at;
  if (i >= n) return;
  const unsigned lanes = 1u << spread, c0 = s.part * lanes * LOOKUP_U + s.in;
  const long long tok = (long long)tokens[i];
  const bool there = tok >= 0 && (size_t)tok < rows;
  const T* const from = weight + (there ? (size_t)tok * stride : 0);
  T* const to = out + i * pieces * V;
  words<T, V> w[LOOKUP_U];
#pragma unroll
  for (int u = 0; u < LOOKUP_U; ++u)
    if (there && c0 + u * lanes < pieces) w[u] = load_words<T, V>(from + (size_t)(c0 + u * lanes) * V);
#pragma unroll
  for (int u = 0; u < LOOKUP_U; ++u)
    if (c0 + u * lanes < pieces) {
      float f[V];
      if (there) channels(w[u], f);
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = there ? scale * f[v] : 0.f;
      store_words<T, V>(to + (size_t)(c0 + u * lanes) * V, to_words<T, V>(f));
    }
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

// how many of keys[0, n) are below `key`, by a whole warp: 32 probes a round trip
__device__ __forceinline__ size_t warp_lower_bound(const unsigned* keys, size_t n, unsigned key) {
  size_t lo = 0, hi = n;
  const unsigned lane = threadIdx.x % 32;
  while (hi - lo > 32) {
    const size_t step = (hi - lo + 32) / 33, at = lo + (lane + 1) * step - 1;      // 32 probes part it into 33
    const unsigned below = __popc(__ballot_sync(tb200::FULL_MASK, at < hi && keys[at] < key));
    const size_t next = lo + below * step;
    if (lo + (below + 1) * step - 1 < hi) hi = lo + (below + 1) * step - 1;
    lo = next;
  }
  return lo + __popc(__ballot_sync(tb200::FULL_MASK, lo + lane < hi && keys[lo + lane] < key));
}

// The gradient, over the tokens' places in the order of the tokens.
//   sums     A CTA takes a chunk of neighbouring places and a run of columns, a thread V of them: it adds up the rows of its chunk run by run (a run:
//            places of the same token), GRAD_U rows requested ahead.  A run that lies in the chunk becomes a row of the result; what a run has in a chunk
//            that it enters or leaves goes to two rows of 32-bit sums a chunk.
//   zeros    Further CTAs of the same launch clear the rows whose token does not occur, GRAD_ZERO rows each.
//   joins    Where a run leaves the chunk in which it begins, its parts are added up, in order.
// So every row of dout is read once, every row of the result is written once, and the order of all sums is the places'.
constexpr int GRAD_U = 8;
constexpr int GRAD_BLOCK = 256;
constexpr unsigned GRAD_ZERO = 32;

struct grad_shape {
  unsigned chunk;        // places of a chunk
  size_t chunks;
  unsigned spread;       // 2^spread threads take columns of a chunk side by side
  unsigned parts;        // how many such groups take all columns
};

template <class O, int V> __device__ __forceinline__ void write_sum(O* to, const float (&sum)[V], float scale, bool accumulate) {
  float f[V];
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = sum[v] * scale;
  if (accumulate) {
    float old[V];
    channels(load_words<O, V>(to), old);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] += old[v];
  }
  store_words<O, V>(to, to_words<O, V>(f));
}
// rows of sums: in 16-byte pieces where V is a multiple of four (dim is one of V then)
template <int V> __device__ __forceinline__ void write_part(float* to, const float (&sum)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int v = 0; v < V; v += 4) *reinterpret_cast<float4*>(to + v) = make_float4(sum[v], sum[v + 1], sum[v + 2], sum[v + 3]);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) to[v] = sum[v];
  }
}
template <int V> __device__ __forceinline__ void read_part(const float* from, float (&sum)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int v = 0; v < V; v += 4) {
      const float4 f = *reinterpret_cast<const float4*>(from + v);
      sum[v] = f.x; sum[v + 1] = f.y; sum[v + 2] = f.z; sum[v + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = from[v];
  }
}

template <class T, class O, int V>
__global__ void __launch_bounds__(GRAD_BLOCK) embedding_grad_kernel(const T* __restrict__ dout, size_t stride, const unsigned* __restrict__ keys, const unsigned* __restrict__ positions,
                                                                  size_t n, unsigned rows, unsigned pieces, grad_shape shape, float scale, bool accumulate, unsigned zero_blocks,
                                                                  O* __restrict__ out, float* __restrict__ partial, const tb200::ws_header* hdr) {
  const size_t dim = (size_t)pieces * V;
  if (hdr->error) {      // the sort's waits ran out
    for (size_t i = (size_t)blockIdx.x * GRAD_BLOCK + threadIdx.x; i < rows * dim; i += (size_t)gridDim.x * GRAD_BLOCK) out[i] = from_f32<O>(__int_as_float(0x7fffffff));
    return;
  }
  if (blockIdx.x < zero_blocks) {
    __shared__ unsigned present;
    const unsigned first = blockIdx.x * GRAD_ZERO, count = rows - first < GRAD_ZERO ? rows - first : GRAD_ZERO;
    if (threadIdx.x < 32) {
      unsigned mine = 0;
      bool more = true;
      for (size_t i = warp_lower_bound(keys, n, first) + threadIdx.x; more; i += 32) {
        const unsigned key = i < n ? keys[i] : ~0u;
        if (key < first + count) mine |= 1u << (key - first);
        more = __all_sync(tb200::FULL_MASK, key < first + count);
      }
      mine = __reduce_or_sync(tb200::FULL_MASK, mine);
      if (threadIdx.x == 0) present = mine;
    }
    __syncthreads();
    float none[V];
#pragma unroll
    for (int v = 0; v < V; ++v) none[v] = 0.f;
    for (unsigned r = 0; r < count; ++r)
      if (!(present >> r & 1))
        for (unsigned c = threadIdx.x; c < pieces; c += GRAD_BLOCK) store_words<O, V>(out + (size_t)(first + r) * dim + (size_t)c * V, to_words<O, V>(none));
    return;
  }
  const share mine = share_of((size_t)(blockIdx.x - zero_blocks) * GRAD_BLOCK + threadIdx.x, shape.spread, shape.parts);
  const size_t chunk = mine.at;
  const unsigned c = (mine.part << shape.spread) + mine.in;
  if (chunk >= shape.chunks || c >= pieces) return;
  const size_t begin = chunk * shape.chunk, end = begin + shape.chunk < n ? begin + shape.chunk : n;
  const T* const from = dout + (size_t)c * V;
  bool entered = begin > 0 && keys[begin - 1] == keys[begin];
  unsigned key = keys[begin];
  float sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) sum[v] = 0.f;
  auto finish = [&](bool leaves) {
    if (key < rows) {
      if (entered) write_part<V>(partial + (2 * chunk) * dim + (size_t)c * V, sum);
      else if (leaves) write_part<V>(partial + (2 * chunk + 1) * dim + (size_t)c * V, sum);
      else write_sum<O, V>(out + (size_t)key * dim + (size_t)c * V, sum, scale, accumulate);
    }
    entered = false;
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = 0.f;
  };
  for (size_t i0 = begin; i0 < end; i0 += GRAD_U) {
    words<T, V> r[GRAD_U];
    unsigned k[GRAD_U];
#pragma unroll
    for (int u = 0; u < GRAD_U; ++u) {
      k[u] = i0 + u < end ? keys[i0 + u] : rows;
      if (k[u] < rows) r[u] = load_words<T, V>(from + (size_t)positions[i0 + u] * stride);
    }
#pragma unroll
    for (int u = 0; u < GRAD_U; ++u) {
      if (i0 + u >= end) break;
      if (k[u] != key) { finish(false); key = k[u]; }
      if (key < rows) {
        float f[V];
        channels(r[u], f);
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] += f[v];
      }
    }
  }
  finish(end < n && keys[end] == key);
}

template <class O, int V>
__global__ void __launch_bounds__(GRAD_BLOCK) embedding_grad_join_kernel(const unsigned* __restrict__ keys, size_t n, unsigned rows, unsigned pieces, grad_shape shape, float scale,
                                                                       bool accumulate, O* __restrict__ out, const float* __restrict__ partial, const tb200::ws_header* hdr) {
  tb200::grid_dependency_wait();
  if (hdr->error) return;
  const size_t dim = (size_t)pieces * V;
  const share mine = share_of((size_t)blockIdx.x * GRAD_BLOCK + threadIdx.x, shape.spread, shape.parts);
  const size_t chunk = mine.at;
  const unsigned c = (mine.part << shape.spread) + mine.in;
  if (chunk + 1 >= shape.chunks || c >= pieces) return;
  const size_t begin = chunk * shape.chunk, end = begin + shape.chunk;
  const unsigned key = keys[end - 1];
  if (key >= rows || keys[end] != key) return;                                              // no run leaves this chunk
  if (begin > 0 && keys[begin] == key && keys[begin - 1] == key) return;                    // one does that has begun earlier
  size_t lo = chunk + 1, hi = shape.chunks;            // how many chunks begin with this token: those behind this one up to lo
  while (lo < hi) { const size_t mid = (lo + hi) >> 1; if (keys[mid * shape.chunk] == key) lo = mid + 1; else hi = mid; }
  float sum[V];
  const float* p = partial + (size_t)c * V;
  read_part<V>(p + (2 * chunk + 1) * dim, sum);
  constexpr int AHEAD = V > 1 ? 4 : GRAD_U;
  for (size_t q = chunk + 1; q < lo; q += AHEAD) {
    float f[AHEAD][V];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (q + u < lo) read_part<V>(p + 2 * (q + u) * dim, f[u]);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (q + u < lo) {
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] += f[u][v];
      }
  }
  write_sum<O, V>(out + (size_t)key * dim + (size_t)c * V, sum, scale, accumulate);
}

// Chunks of 64 places, smaller ones (down to 8) while fewer than a thousand threads a SM would have work.
constexpr size_t GRAD_THREADS = 148 * 1024;
grad_shape grad_shape_of(size_t n, size_t pieces) {
  grad_shape s;
  s.spread = spread_of(pieces, 8);
  s.parts = (unsigned)((pieces + (size_t(1) << s.spread) - 1) >> s.spread);
  s.chunk = 64;
  while (s.chunk > 8 && ((n + s.chunk - 1) / s.chunk * s.parts << s.spread) < GRAD_THREADS) s.chunk /= 2;
  s.chunks = (n + s.chunk - 1) / s.chunk;
  return s;
}

// the workspace: the sort's, then keys, positions and the sort's other halves, then the chunks' sums
struct grad_layout {
  size_t array, sort, partial, need;
  grad_layout(size_t n, size_t dim) {
    array = tb200::align_up(n * 4, 256);
    sort = tb200::align_up(tb200::radix_workspace_bytes<4, 4>(n), 256);
    partial = sort + 4 * array;
    // as many chunks as there can be, whatever the pieces: of 8 places, or 64 and, where they are smaller, at most GRAD_THREADS to the half of them
    const grad_shape s = grad_shape_of(n, (dim + 7) / 8);
    const size_t most = n / 64 + 2 * GRAD_THREADS / ((size_t)s.parts << s.spread) + 2, chunks = (n + 7) / 8 < most ? (n + 7) / 8 : most;
    need = partial + 2 * chunks * dim * 4;
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
      if (!d_tokens || !d_out || (rows && !d_weight) || weight_stride < dim || n >= (1ull << 31) || dim >= (1ull << 31)) return ERR_INVALID;
      auto go = [&](auto vv) -> int {
        constexpr int V = decltype(vv)::value;
        const unsigned pieces = (unsigned)(dim / V), spread = spread_of((pieces + LOOKUP_U - 1) / LOOKUP_U, 5), parts = (unsigned)(((size_t)pieces + (LOOKUP_U << spread) - 1) / (LOOKUP_U << spread));
        const size_t grid = (((n * parts) << spread) + 255) / 256;
        if (grid > 0x7fffffffull) return ERR_INVALID;
        embedding_kernel<T, V, I><<<(unsigned)grid, 256, 0, stream>>>(static_cast<const T*>(d_weight), rows, weight_stride, static_cast<const I*>(d_tokens), n, pieces, parts, spread, scale,
                                                                    static_cast<T*>(d_out));
        return (int)cudaGetLastError();
      };
      if (in_16_bytes(d_weight, dim, weight_stride, sizeof(T)) && in_16_bytes(d_out, dim, dim, sizeof(T))) return go(std::integral_constant<int, 16 / sizeof(T)>());
      return go(std::integral_constant<int, 1>());
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
        const grad_layout lay(n, dim);
        int rc;
        if (workspace_gate(d_ws, ws_bytes, lay.need, rc)) return rc;
        if (rows == 0 || dim == 0) return 0;
        if (!d_out || (n && (!d_dout || !d_tokens)) || dout_stride < dim || dim >= (1ull << 31)) return ERR_INVALID;
        char* const base = static_cast<char*>(d_ws);
        unsigned* const keys = reinterpret_cast<unsigned*>(base + lay.sort);
        unsigned* const positions = reinterpret_cast<unsigned*>(base + lay.sort + 2 * lay.array);
        float* const partial = reinterpret_cast<float*>(base + lay.partial);
        if (n) token_keys_kernel<I><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(static_cast<const I*>(d_tokens), n, (unsigned)rows, keys, positions);
        tb200::key_coding coding;
        coding.kind = tb200::KEY_UNSIGNED;
        coding.descending = 0;
        int bits = 8;
        while (bits < 32 && (rows >> bits)) bits += 8;      // the largest key is `rows`
        const cudaError_t e = tb200::radix_sort_async<uint32_t, uint32_t, true>(keys, keys + lay.array / 4, positions, positions + lay.array / 4, n, coding, 0, bits, d_ws, stream);
        if (e != cudaSuccess) return (int)e;
        auto go = [&](auto vv) -> int {
          constexpr int V = decltype(vv)::value;
          const unsigned pieces = (unsigned)(dim / V);
          const grad_shape shape = grad_shape_of(n, pieces);
          const tb200::ws_header* hdr = static_cast<const tb200::ws_header*>(d_ws);
          const unsigned zero_blocks = accumulate ? 0u : (unsigned)((rows + GRAD_ZERO - 1) / GRAD_ZERO);
          const size_t grid = ((shape.chunks * shape.parts << shape.spread) + GRAD_BLOCK - 1) / GRAD_BLOCK;
          if (grid + zero_blocks > 0x7fffffffull) return ERR_INVALID;
          if (grid + zero_blocks == 0) return 0;
          embedding_grad_kernel<T, O, V><<<(unsigned)(grid + zero_blocks), GRAD_BLOCK, 0, stream>>>(static_cast<const T*>(d_dout), dout_stride, keys, positions, n, (unsigned)rows, pieces,
                                                                                                shape, scale, accumulate != 0, zero_blocks, static_cast<O*>(d_out), partial, hdr);
          const cudaError_t e = cudaGetLastError();
          if (e != cudaSuccess || shape.chunks < 2) return (int)e;
          return (int)tb200::launch_after(embedding_grad_join_kernel<O, V>, grid, GRAD_BLOCK, 0, stream, keys, n, (unsigned)rows, pieces, shape, scale, accumulate != 0,
                                          static_cast<O*>(d_out), partial, hdr);
        };
        // pieces of 16 bytes of the wider of the two types, at most 8 channels: both sides are aligned to theirs then
        constexpr int WIDE = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
        if (in_16_bytes(d_dout, dim, dout_stride, sizeof(T)) && in_16_bytes(d_out, dim, dim, sizeof(O))) return go(std::integral_constant<int, WIDE>());
        return go(std::integral_constant<int, 1>());
      });
    });
  });
}
