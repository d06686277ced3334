// C ABI: tb200_expert_dispatch, tb200_expert_combine and tb200_expert_combine_grad.
#include "abi_rows.cuh"

using namespace tb200_abi;
using namespace tb200_rows;

namespace {
constexpr int MOST_EXPERTS = 1024;
constexpr int MOST_CHOICES = 32;
constexpr int DISPATCH_BLOCK = 1024;
constexpr int SMALL_BLOCK = 256;
static_assert((2 + SMALL_BLOCK / 32) * MOST_EXPERTS * 4 <= 40 * 1024, "the small block's dynamic shared memory, beside what it has besides");
constexpr unsigned COUNT_HERE = 8192;      // up to so many assignments every CTA counts them all itself

template <class I> __device__ __forceinline__ unsigned expert_of(const I* ids, size_t i, unsigned experts) {      // `experts` for an id that is none
  const long long e = (long long)ids[i];
  return e >= 0 && e < (long long)experts ? (unsigned)e : experts;
}

// table[block][expert]: how many assignments of the block's tokens go there
template <class I>
__global__ void __launch_bounds__(DISPATCH_BLOCK) expert_count_kernel(const I* ids, size_t n, unsigned choices, unsigned experts, unsigned* table) {
  __shared__ unsigned count[MOST_EXPERTS];
  for (unsigned e = threadIdx.x; e < experts; e += DISPATCH_BLOCK) count[e] = 0;
  __syncthreads();
  const size_t per = (n + gridDim.x - 1) / gridDim.x, first = blockIdx.x * per < n ? blockIdx.x * per : n, stop = first + per < n ? first + per : n;
  for (size_t i = first * choices + threadIdx.x; i < stop * choices; i += DISPATCH_BLOCK) {
    const unsigned e = expert_of(ids, i, experts);
    if (e < experts) atomicAdd(&count[e], 1u);
  }
  __syncthreads();
  for (unsigned e = threadIdx.x; e < experts; e += DISPATCH_BLOCK) table[(size_t)blockIdx.x * experts + e] = count[e];
  tb200::grid_dependents_launch();
}

// A stable counting sort of the assignments and the rows' way to their places, in one kernel.  A CTA has the assignments of neighbouring tokens.
// It adds up, by expert, all assignments and those before its own (from the blocks' counts, or from the ids while they are few), ranks its own
// ones warp by warp, and copies each of its tokens' rows to its places: a row is read once and written as often as it goes somewhere.
// Bound by the bytes of the rows, most of them scattered writes: 16384 bf16 rows of 2048 to 8 of 128 experts take 123 us (4900 GB/s), of which counting and
// ranking are the first 9.  Rows in the order of their places, gathered by their sources, take 144: each is read eight times then.
// (table is written while this kernel may already be resident: not __restrict__, which would allow loads that are for data that does not change.)
template <class V, class I, bool COUNTED>
__global__ void __launch_bounds__(DISPATCH_BLOCK) expert_dispatch_kernel(const V* __restrict__ x, size_t xs, const I* __restrict__ ids, size_t n, unsigned choices, unsigned experts,
                                                                       size_t pieces, unsigned spread, V* __restrict__ rows, int* slots, int* sources, int* offsets,
                                                                       const unsigned* table, tb200::ws_header* hdr) {
  extern __shared__ unsigned raw[];
  const unsigned warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  unsigned* const total = raw;                    // [experts]
  unsigned* const start = total + experts;        // [experts]: of this CTA's assignments, first how many come before them
  unsigned* const at = start + experts;           // [warps][experts]
  __shared__ unsigned kept;
  const size_t m = n * choices;
  const size_t per = (n + gridDim.x - 1) / gridDim.x, first = blockIdx.x * per < n ? blockIdx.x * per : n, stop = first + per < n ? first + per : n;
  const size_t i0 = first * choices, i1 = stop * choices;
  for (unsigned e = threadIdx.x; e < (2 + warps) * experts; e += blockDim.x) raw[e] = 0;
  __syncthreads();
  if (COUNTED) {
    tb200::grid_dependency_wait();
    // a column of the table is one thread's, or several threads' that take its rows in turn
    const unsigned turns = blockDim.x / experts > 0 ? blockDim.x / experts : 1, e = threadIdx.x % experts, turn = threadIdx.x / experts;
    if (turn < turns && threadIdx.x < turns * experts) {
      unsigned all = 0, before = 0;
#pragma unroll 8
      for (unsigned r = turn; r < gridDim.x; r += turns) {
        const unsigned c = table[(size_t)r * experts + e];
        all += c;
        before += r < blockIdx.x ? c : 0;
      }
      if (all) atomicAdd(&total[e], all);
      if (before) atomicAdd(&start[e], before);
    }
  } else {
    for (size_t i = threadIdx.x; i < m; i += blockDim.x) {
      const unsigned e = expert_of(ids, i, experts);
      if (e < experts) {
        atomicAdd(&total[e], 1u);
        if (i < i0) atomicAdd(&start[e], 1u);
      }
    }
  }
  // this warp's assignments: neighbouring ones
  const size_t share = ((i1 - i0 + warps - 1) / warps + 31) / 32 * 32;
  const size_t w0 = i0 + warp * share < i1 ? i0 + warp * share : i1, w1 = w0 + share < i1 ? w0 + share : i1;
  unsigned* const own = at + warp * experts;
  for (size_t i = w0 + lane; i < w1; i += 32) {
    const unsigned e = expert_of(ids, i, experts);
    if (e < experts) atomicAdd(&own[e], 1u);
  }
  __syncthreads();
  if (warp == 0) {
    unsigned sum = 0;
    for (unsigned base = 0; base < experts; base += 32) {
      const unsigned e = base + lane, c = e < experts ? total[e] : 0;
      const unsigned inclusive = tb200::warp_inclusive_scan(c, tb200::plus_op());
      if (e < experts) {
        const unsigned o = sum + inclusive - c;
        start[e] += o;
        if (blockIdx.x == 0) offsets[e] = (int)o;
      }
      sum += __shfl_sync(tb200::FULL_MASK, inclusive, 31);
    }
    if (lane == 0) {
      kept = sum;
      if (blockIdx.x == 0) { offsets[experts] = (int)sum; hdr->error = 0; }      // nothing here waits
    }
  }
  __syncthreads();
  for (unsigned e = threadIdx.x; e < experts; e += blockDim.x) {
    unsigned next = start[e];
    for (unsigned w = 0; w < warps; ++w) { const unsigned c = at[w * experts + e]; at[w * experts + e] = next; next += c; }
  }
  __syncthreads();
  for (size_t base = w0; base < w1; base += 32) {
    const size_t i = base + lane;
    const unsigned e = i < w1 ? expert_of(ids, i, experts) : experts;
    const unsigned same = __match_any_sync(tb200::FULL_MASK, e);
    const unsigned before = __popc(same & ((1u << lane) - 1));
    unsigned place = 0;
    if (e < experts) place = own[e] + before;
    __syncwarp();
    if (e < experts) {
      if (before == 0) own[e] += __popc(same);
      slots[i] = (int)place;
      sources[place] = (int)i;
    } else if (i < w1) {
      slots[i] = -1;
    }
    __syncwarp();
  }
  __syncthreads();
  constexpr int U = 8;
  const unsigned g = 1u << spread, group = threadIdx.x / g, groups = blockDim.x / g, in = threadIdx.x % g;
  for (size_t token = first + group; token < stop; token += groups) {
    const V* const from = x + token * xs;
    for (size_t c0 = in; c0 < pieces; c0 += (size_t)g * U) {
      V v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + (size_t)u * g < pieces) v[u] = from[c0 + (size_t)u * g];
      for (unsigned k = 0; k < choices; ++k) {
        const int place = slots[token * choices + k];
        if (place < 0) continue;
        V* const to = rows + (size_t)place * pieces;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c0 + (size_t)u * g < pieces) to[c0 + (size_t)u * g] = v[u];
      }
    }
  }
  // rows that nothing goes to
  for (size_t row = (size_t)kept + (size_t)blockIdx.x * groups + group; row < m; row += (size_t)gridDim.x * groups) {
    if (in == 0) sources[row] = -1;
    V* const to = rows + row * pieces;
    for (size_t c = in; c < pieces; c += g) to[c] = V{};
  }
}

// A thread has up to U pieces of a token's result, and requests those of K of its rows at a time.  ALL: K rows are all there are, so that no sums have
// to be held while rows are on their way: few registers, many reads in flight.  Bound by the bytes of the rows: 8191 f16 rows of 4096, the sums of two, take
// 33 us, of which 31 are bytes.
template <class T, int V, bool WEIGHTED, int K, int U, bool ALL>
__global__ void __launch_bounds__(256) expert_combine_kernel(const T* __restrict__ rows, size_t rs, unsigned m, const int* __restrict__ slots, const float* __restrict__ weights,
                                                             size_t n, unsigned choices, unsigned pieces, unsigned spread, unsigned parts, T* __restrict__ out) {
  const share s = share_of((size_t)blockIdx.x * 256 + threadIdx.x, spread, parts);
  const size_t token = s.at;
  if (token >= n) return;
  const unsigned lanes = 1u << spread, c0 = s.part * lanes * U + s.in;
  const int* const at = slots + token * choices;
  T* const to = out + token * pieces * V;
  float sum[ALL ? 1 : U][V];
#pragma unroll
  for (int u = 0; u < (ALL ? 1 : U); ++u)
#pragma unroll
    for (int v = 0; v < V; ++v) sum[u][v] = 0.f;
  for (unsigned k0 = 0; k0 < (ALL ? 1 : choices); k0 += K) {
    words<T, V> r[K][U];
    bool there[K];
#pragma unroll
    for (unsigned j = 0; j < K; ++j) {
      const int place = k0 + j < choices ? at[k0 + j] : -1;
      there[j] = (unsigned)place < m;
      const T* const from = rows + (there[j] ? (size_t)place * rs : 0);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (there[j] && c0 + u * lanes < pieces) r[j][u] = load_words<T, V>(from + (size_t)(c0 + u * lanes) * V);
    }
    float w[K];
#pragma unroll
    for (unsigned j = 0; j < K; ++j) w[j] = WEIGHTED && there[j] ? weights[token * choices + k0 + j] : 1.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float (&t)[V] = sum[ALL ? 0 : u];
      if (ALL) {
#pragma unroll
        for (int v = 0; v < V; ++v) t[v] = 0.f;
      }
#pragma unroll
      for (unsigned j = 0; j < K; ++j)
        if (there[j]) {
          float f[V];
          channels(r[j][u], f);
#pragma unroll
          for (int v = 0; v < V; ++v) t[v] = WEIGHTED ? fmaf(w[j], f[v], t[v]) : t[v] + f[v];
        }
      if (ALL && c0 + u * lanes < pieces) store_words<T, V>(to + (size_t)(c0 + u * lanes) * V, to_words<T, V>(t));
    }
  }
  if (!ALL) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * lanes < pieces) store_words<T, V>(to + (size_t)(c0 + u * lanes) * V, to_words<T, V>(sum[ALL ? 0 : u]));
  }
}

// 2^spread lanes a token (WARP: 32, known beforehand, where the rows are long enough): its row of dout stays in registers (while it fits) against the rows of all its choices, each
// read and written once.  Bound by the bytes of the rows: 16384 bf16 rows of 2048 with six choices take 135 us, of which 131 are bytes.
template <class T, int V, bool WARP>
__global__ void __launch_bounds__(256) expert_combine_grad_kernel(const T* __restrict__ dout, size_t ds, const T* __restrict__ rows, size_t rs, size_t m, const int* __restrict__ slots,
                                                                  const float* __restrict__ weights, const int* __restrict__ end, size_t n, unsigned choices, size_t pieces,
                                                                  unsigned lanes_log, T* __restrict__ drows, float* __restrict__ dweights) {
  constexpr int U = 8;
  const unsigned spread = WARP ? 5 : lanes_log, lanes = 1u << spread, in = threadIdx.x & (lanes - 1);
  const size_t groups = ((size_t)gridDim.x * 256) >> spread, index = ((size_t)blockIdx.x * 256 + threadIdx.x) >> spread;
  const size_t dim = pieces * V, rounds = (n + groups - 1) / groups;
  for (size_t round = 0; round < rounds; ++round) {      // the same for all groups of a warp
    const size_t token = index + round * groups;
    const bool there = token < n;
    const T* const d = dout + (there ? token : 0) * ds;
    words<T, V> held[U];
    auto take = [&](size_t c0) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * lanes < pieces) held[u] = load_words<T, V>(d + (c0 + u * lanes) * V);
    };
    if (there && pieces <= (size_t)U * lanes) take(in);
    for (unsigned k = 0; k < choices; ++k) {
      const int place = there ? slots[token * choices + k] : -1;
      float dot = 0.f;
      if ((unsigned)place < m) {
        const float w = weights[token * choices + k];
        const T* const r = rows + (size_t)place * rs;
        T* const to = drows + (size_t)place * dim;
        for (size_t c0 = in; c0 < pieces; c0 += (size_t)U * lanes) {
          words<T, V> v[U];
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + u * lanes < pieces) v[u] = load_words<T, V>(r + (c0 + u * lanes) * V);
          if (pieces > (size_t)U * lanes) take(c0);
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (c0 + u * lanes < pieces) {
              float a[V], b[V];
              channels(held[u], a);
              channels(v[u], b);
#pragma unroll
              for (int i = 0; i < V; ++i) { dot = fmaf(a[i], b[i], dot); a[i] *= w; }
              store_words<T, V>(to + (c0 + u * lanes) * V, to_words<T, V>(a));
            }
        }
      }
#pragma unroll
      for (unsigned o = 16; o; o >>= 1)
        if (WARP || o < lanes) dot += __shfl_xor_sync(tb200::FULL_MASK, dot, o);
      if (there && in == 0) dweights[token * choices + k] = dot;
    }
  }
  float none[V];
#pragma unroll
  for (int v = 0; v < V; ++v) none[v] = 0.f;
  const int kept = *end;
  for (size_t row = (kept > 0 ? (size_t)kept : 0) + index; row < m; row += groups)
    for (size_t c = in; c < pieces; c += lanes) store_words<T, V>(drows + row * dim + c * V, to_words<T, V>(none));
}

// what every one of these calls needs of its sizes: flat assignments and rows are counted in 31 bits
bool sizes_fit(size_t n, size_t choices) { return choices >= 1 && choices <= (size_t)MOST_CHOICES && n <= 0x7fffffffull / choices / 2; }

unsigned dispatch_grid(size_t n) { const size_t sms = (size_t)tb200::current_device_info().sm_count; return (unsigned)(n < sms ? (n ? n : 1) : sms); }
size_t dispatch_workspace(size_t n, size_t choices, size_t experts) {
  return sizeof(tb200::ws_header) + (n * choices > COUNT_HERE ? (size_t)dispatch_grid(n) * experts * 4 : 0);
}
}  // namespace

TB200_API int tb200_expert_dispatch(const void* d_x, size_t x_stride, const void* d_experts, int expert_t, size_t n, size_t choices, size_t num_experts, size_t dim, int t,
                                    void* d_rows, int* d_slots, int* d_sources, int* d_offsets, void* d_ws, size_t* ws_bytes, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    return by_index_dtype(expert_t, [&](auto iv) -> int {
      using I = decltype(iv);
      if (!sizes_fit(n, choices) || num_experts < 1 || num_experts > (size_t)MOST_EXPERTS) return ERR_INVALID;
      int rc;
      if (workspace_gate(d_ws, ws_bytes, dispatch_workspace(n, choices, num_experts), rc)) return rc;
      const size_t m = n * choices;
      if (!d_offsets || (m && (!d_experts || !d_slots || !d_sources || (dim && (!d_x || !d_rows)))) || x_stride < dim) return ERR_INVALID;
      const unsigned experts = (unsigned)num_experts, grid = dispatch_grid(n);
      const bool counted = m > COUNT_HERE;
      unsigned* const table = reinterpret_cast<unsigned*>(static_cast<char*>(d_ws) + sizeof(tb200::ws_header));
      auto go = [&](auto vv, auto cv) -> int {
        using V = decltype(vv);
        constexpr bool COUNTED = decltype(cv)::value;
        const int block = COUNTED ? DISPATCH_BLOCK : SMALL_BLOCK;
        const size_t smem = (2 + (size_t)block / 32) * experts * 4;
        auto kernel = expert_dispatch_kernel<V, I, COUNTED>;
        if (COUNTED) {      // (the smaller block needs no more than any kernel may have)
          // the most that any call needs: the limit is the kernel's, and calls in other threads may lie between this line and the launch
          const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (2 + DISPATCH_BLOCK / 32) * MOST_EXPERTS * 4);
          if (e != cudaSuccess) return (int)e;
          expert_count_kernel<I><<<grid, DISPATCH_BLOCK, 0, stream>>>(static_cast<const I*>(d_experts), n, (unsigned)choices, experts, table);
        }
        const size_t scale = sizeof(V) / sizeof(T);
        if (COUNTED)      // begins while the blocks are still counted, and waits for that
          return (int)tb200::launch_after(kernel, grid, block, smem, stream, static_cast<const V*>(d_x), x_stride / scale, static_cast<const I*>(d_experts), n, (unsigned)choices, experts,
                                          dim / scale, spread_of(dim / scale, 5), static_cast<V*>(d_rows), d_slots, d_sources, d_offsets, table,
                                          static_cast<tb200::ws_header*>(d_ws));
        kernel<<<grid, block, smem, stream>>>(static_cast<const V*>(d_x), x_stride / scale, static_cast<const I*>(d_experts), n, (unsigned)choices, experts, dim / scale,
                                              spread_of(dim / scale, 5), static_cast<V*>(d_rows), d_slots, d_sources, d_offsets, table, static_cast<tb200::ws_header*>(d_ws));
        return (int)cudaGetLastError();
      };
      auto with = [&](auto vv) -> int { return counted ? go(vv, std::true_type()) : go(vv, std::false_type()); };
      if (in_16_bytes(d_x, dim, x_stride, sizeof(T)) && in_16_bytes(d_rows, dim, dim, sizeof(T))) return with(uint4());
      if constexpr (sizeof(T) == 4) return with(unsigned());
      else return with((unsigned short)0);
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
    auto go = [&](auto vv, auto wv) -> int {
      constexpr int V = decltype(vv)::value;
      if (dim >= (1ull << 31)) return ERR_INVALID;
      const unsigned pieces = (unsigned)(dim / V);
      auto run = [&](auto kk, auto uu, auto all) -> int {
        constexpr int K = decltype(kk)::value, U = decltype(uu)::value;
        const unsigned spread = spread_of((pieces + U - 1) / U, 5), parts = (unsigned)(((size_t)pieces + (U << spread) - 1) / (U << spread));
        const size_t grid = (((n * parts) << spread) + 255) / 256;
        if (grid > 0x7fffffffull) return ERR_INVALID;
        expert_combine_kernel<T, V, decltype(wv)::value, K, U, decltype(all)::value><<<(unsigned)grid, 256, 0, stream>>>(
            static_cast<const T*>(d_rows), rows_stride, (unsigned)(n * choices), d_slots, d_weights, n, (unsigned)choices, pieces, spread, parts, static_cast<T*>(d_out));
        return (int)cudaGetLastError();
      };
      using std::integral_constant;
      // 16-byte pieces, four to eight reads a thread.  8191 x 2 f16 rows of 4096: 34 us (two rows at a time with their sums held: 39, eight reads with four sums: 45);
      // 8192 x 8 bf16 rows of 2048: 50 (two at a time: 52); 16384 x 1 of 4096: 45 (62).  Channel by channel two of eight rows at a time are faster than all of
      // them: 8192 x 4 bf16 rows of 1501: 42 us against 72 (eight pieces a thread; four: 52).
      if constexpr (V > 1) {
        if (choices == 1) return run(integral_constant<int, 1>(), integral_constant<int, 4>(), std::true_type());
        if (choices == 2) return run(integral_constant<int, 2>(), integral_constant<int, 2>(), std::true_type());
        if (choices <= 4) return run(integral_constant<int, 4>(), integral_constant<int, 2>(), std::true_type());
        if (choices <= 8) return run(integral_constant<int, 8>(), integral_constant<int, 1>(), std::true_type());
        return run(integral_constant<int, 2>(), integral_constant<int, 2>(), std::false_type());
      } else {
        return run(integral_constant<int, 2>(), integral_constant<int, 8>(), std::false_type());
      }
    };
    auto with = [&](auto vv) -> int { return d_weights ? go(vv, std::true_type()) : go(vv, std::false_type()); };
    if (in_16_bytes(d_rows, dim, rows_stride, sizeof(T)) && in_16_bytes(d_out, dim, dim, sizeof(T))) return with(std::integral_constant<int, 16 / sizeof(T)>());
    return with(std::integral_constant<int, 1>());
  });
}

TB200_API int tb200_expert_combine_grad(const void* d_dout, size_t dout_stride, const void* d_rows, size_t rows_stride, const int* d_slots, const float* d_weights,
                                        const int* d_kept, size_t n, size_t choices, size_t dim, int t, void* d_drows, float* d_dweights, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    if (!sizes_fit(n, choices)) return ERR_INVALID;
    if (n == 0) return 0;
    if (!d_slots || !d_weights || !d_kept || !d_dweights || (dim && (!d_dout || !d_rows || !d_drows)) || dout_stride < dim || rows_stride < dim) return ERR_INVALID;
    auto go = [&](auto vv) -> int {
      constexpr int V = decltype(vv)::value;
      const unsigned spread = spread_of(dim / V, 5);
      const size_t most = (size_t)tb200::current_device_info().sm_count * 16, want = ((n << spread) + 255) / 256;
      (spread == 5 ? expert_combine_grad_kernel<T, V, true> : expert_combine_grad_kernel<T, V, false>)<<<(unsigned)(want < most ? want : most), 256, 0, stream>>>(static_cast<const T*>(d_dout), dout_stride, static_cast<const T*>(d_rows), rows_stride,
                                                                                              n * choices, d_slots, d_weights, d_kept, n, (unsigned)choices, dim / V, spread,
                                                                                              static_cast<T*>(d_drows), d_dweights);
      return (int)cudaGetLastError();
    };
    if (in_16_bytes(d_dout, dim, dout_stride, sizeof(T)) && in_16_bytes(d_rows, dim, rows_stride, sizeof(T)) && in_16_bytes(d_drows, dim, dim, sizeof(T)))
      return go(std::integral_constant<int, 16 / sizeof(T)>());
    return go(std::integral_constant<int, 1>());
  });
}
