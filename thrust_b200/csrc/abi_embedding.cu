// C ABI: tb200_embedding and tb200_embedding_grad.
#include "abi_rows.cuh"
#include "thrust_b200/radix_sort.cuh"

using namespace tb200_abi;
using namespace tb200_rows;

namespace {
// out[i] = scale * weight[tokens[i]].  2^spread lanes take up to LOOKUP_U pieces each of a row (`parts` times that make a row): as many random reads
// are in flight per thread.  Bound by the bytes of the rows: 16391 bf16 rows of 4096 from a table of 100003 take 34 us, of which 29 are bytes.
// Channel by channel 16 reads of 32 bits (16391 rows of 2049: 44 us, with four 55) or eight of 16 (with 16 57, with four 53)
constexpr int lookup_u(int v, size_t bytes) { return v > 1 ? 4 : bytes == 4 ? 16 : 8; }
template <class T, int V, class I>
__global__ void __launch_bounds__(256) embedding_kernel(const T* __restrict__ weight, size_t rows, size_t stride, const I* __restrict__ tokens, size_t n, unsigned pieces, unsigned parts,
                                                        unsigned spread, float scale, T* __restrict__ out) {
  constexpr int LOOKUP_U = lookup_u(V, sizeof(T));
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

// keys: the token, or `rows` for one that is no row; positions 0, 1, ...; and the lists of long runs are empty
template <class I>
__global__ void __launch_bounds__(256) token_keys_kernel(const I* tokens, size_t n, unsigned rows, unsigned* keys, unsigned* positions, unsigned* counts) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i < 2) counts[i] = 0;
  if (i >= n) return;
  const long long tok = (long long)tokens[i];
  keys[i] = tok >= 0 && tok < (long long)rows ? (unsigned)tok : rows;
  positions[i] = (unsigned)i;
}

// The same places, sorted, where there are few: the rank of a place is the number of places whose key is smaller, or the same and further in front.  A CTA has
// all keys in shared memory, its lanes P places each and its warps a share of the keys each: P = 1 while that makes a CTA a SM at most, so that no SM has twice
// the others' work.  Bound by n * n additions; one kernel instead of the sort's two.  A whole gradient (bf16 rows of 1000 added to f32) takes 18 us instead of 26
// for 4099 places and 30 instead of 33 for 8192; for 10000 it would take 40 instead of 34.
constexpr unsigned PLACE_MOST = 8192, PLACE_BLOCK = 1024;
// count + (not_key's key < limit): the sum limit + ~key carries then
__device__ __forceinline__ unsigned count_below(unsigned count, unsigned not_key, unsigned limit) {
  asm("{.reg .u32 t; add.cc.u32 t, %1, %2; addc.u32 %0, %0, 0;}" : "+r"(count) : "r"(limit), "r"(not_key));
  return count;
}
template <int P, class I>
__global__ void __launch_bounds__(PLACE_BLOCK) place_kernel(const I* tokens, unsigned n, unsigned rows, unsigned* keys, unsigned* positions, unsigned* counts, tb200::ws_header* hdr) {
  __shared__ uint4 all[PLACE_MOST / 4];
  __shared__ unsigned rank[32 * P];
  tb200::grid_dependents_launch();
  if (blockIdx.x == 0 && threadIdx.x < 2) counts[threadIdx.x] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) hdr->error = 0;
  if (threadIdx.x < 32 * P) rank[threadIdx.x] = 0;
  constexpr unsigned WARPS = PLACE_BLOCK / 32;
  const unsigned fours = (n + 3) / 4, share = (fours + WARPS - 1) / WARPS;      // of each warp
  unsigned* const not_key = reinterpret_cast<unsigned*>(all);
#pragma unroll 4
  for (unsigned i = threadIdx.x; i < fours * 4; i += PLACE_BLOCK) {
    const long long tok = i < n ? (long long)tokens[i] : -1;
    not_key[i] = ~(tok >= 0 && tok < (long long)rows ? (unsigned)tok : i < n ? rows : ~0u);      // the largest behind the last one
  }
  __syncthreads();
  const unsigned lane = threadIdx.x % 32, first = blockIdx.x * 32 * P;
  const unsigned from = threadIdx.x / 32 * share, to = from + share < fours ? from + share : fours;
  unsigned mine[P], below[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const unsigned i = first + p * 32 + lane;
    mine[p] = i < n ? ~not_key[i] : 0;
    below[p] = 0;
  }
  auto count = [&](unsigned a, unsigned b, unsigned more) {
#pragma unroll 4
    for (unsigned j = a; j < b; ++j) {
      const uint4 k = all[j];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const unsigned limit = mine[p] + more;
        below[p] = count_below(count_below(count_below(count_below(below[p], k.x, limit), k.y, limit), k.z, limit), k.w, limit);
      }
    }
  };
  const unsigned here = first / 4, behind = here + 8 * P;      // the fours of this CTA's own places
  count(from, to < here ? to : here, 1);
  for (unsigned j = from > here ? from : here; j < to && j < behind; ++j)
#pragma unroll
    for (unsigned u = 0; u < 4; ++u)
#pragma unroll
      for (int p = 0; p < P; ++p) below[p] = count_below(below[p], not_key[j * 4 + u], mine[p] + (j * 4 + u < first + p * 32 + lane));
  count(from > behind ? from : behind, to, 0);
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (from < to) atomicAdd(&rank[p * 32 + lane], below[p]);
  __syncthreads();
  const unsigned i = first + threadIdx.x;
  if (threadIdx.x < 32 * P && i < n) {
    const unsigned at = rank[threadIdx.x];
    keys[at] = ~not_key[i];
    positions[at] = i;
  }
}

// how many of keys[0, n) are below `key`, by a whole warp: 32 probes a round trip
__device__ __forceinline__ size_t warp_lower_bound(const unsigned* keys, size_t n, unsigned key) {
  size_t lo = 0, hi = n;
  const unsigned lane = threadIdx.x % 32;
  while (hi - lo > 32) {
    const size_t step = (hi - lo + 32) / 33, at = lo + (lane + 1) * step - 1;      // 32 probes part it into 33
    const unsigned below = __popc(__ballot_sync(tb200::FULL_MASK, at < hi && keys[at] < key));
    const size_t next = lo + below * step;
    const size_t probe = lo + (below + 1) * step - 1;      // the first one that is not below, if there is one
    if (below < 32 && probe < hi) hi = probe;
    lo = next;
  }
  return lo + __popc(__ballot_sync(tb200::FULL_MASK, lo + lane < hi && keys[lo + lane] < key));
}

// The gradient, over the tokens' places in the order of the tokens.
//   sums     Some threads take a chunk of neighbouring places, V columns each, and add up its rows run by run (a run: places of the same token), GRAD_U
//            rows requested ahead.  A run that begins in a chunk and ends in the next one at the latest is added up there, and the next chunk leaves it out;
//            of a longer one each chunk adds up its own part, into one of two rows of 32-bit sums that it has.
//   zeros    Further CTAs of the same launch clear the rows whose token does not occur, GRAD_ZERO rows each.
//   joins    The parts of a long run are added up, in order.
// So every row of dout is read once, every row of the result is written once, and the order of all sums is the places'.  Bound by the bytes of those rows once
// there are many: of 163 us for 65536 bf16 rows of 2048 and a table of 128000 the sums and zeros are 124 (5900 GB/s); the sort before them takes 24.  Clearing
// the whole result beforehand would write the rows that occur twice.
constexpr int GRAD_U = 8;
constexpr int GRAD_BLOCK = 256;
constexpr unsigned GRAD_ZERO = 32, GRAD_CHUNK = 32;      // rows cleared by a CTA; most places of a chunk
constexpr unsigned GRAD_SPREAD = 4;                        // at least 16 threads a chunk

struct grad_shape {
  unsigned chunk;        // places of a chunk
  size_t chunks;
  unsigned spread;       // 2^spread threads take columns of a chunk side by side
  unsigned parts;        // how many such groups take all columns
};

// zeros from `from` to `to`, by all threads of the CTA: 16 bytes at a time but for the ends (78666 f32 rows of 1273: 77 us, channel by channel 107)
template <class O> __device__ __forceinline__ void clear_stretch(O* from, O* to) {
  O* const inner = reinterpret_cast<O*>((reinterpret_cast<uintptr_t>(from) + 15) & ~(uintptr_t)15);
  O* const last = reinterpret_cast<O*>(reinterpret_cast<uintptr_t>(to) & ~(uintptr_t)15);
  if (inner >= last) {
    for (O* p = from + threadIdx.x; p < to; p += GRAD_BLOCK) *p = from_f32<O>(0.f);
    return;
  }
  for (uint4* p = reinterpret_cast<uint4*>(inner) + threadIdx.x; p < reinterpret_cast<uint4*>(last); p += GRAD_BLOCK) *p = make_uint4(0, 0, 0, 0);
  for (O* p = from + threadIdx.x; p < inner; p += GRAD_BLOCK) *p = from_f32<O>(0.f);
  for (O* p = last + threadIdx.x; p < to; p += GRAD_BLOCK) *p = from_f32<O>(0.f);
}

// What a chunk has to do with the runs at its two ends.
struct run_ends {
  size_t end, stop;          // behind its last place; behind the last place that it may look at
  unsigned first, last;      // the tokens at its ends
  bool entered;              // its first run has begun in an earlier chunk,
  bool skip;                 // and is added up there
  bool extended;             // its last run goes on in the next chunk, and is added up here all the same
  bool leaves;               // its last run begins here and has a part in at least two more chunks
};
__device__ __forceinline__ run_ends run_ends_of(const unsigned* keys, size_t n, size_t chunk, unsigned size) {
  run_ends r;
  const size_t begin = chunk * size;
  r.end = begin + size < n ? begin + size : n;
  const size_t next = r.end + size < n ? r.end + size : n;
  r.first = keys[begin];
  r.last = keys[r.end - 1];
  const unsigned before = begin ? keys[begin - 1] : ~r.first, behind = r.end < n ? keys[r.end] : ~r.last;
  const unsigned previous = begin ? keys[begin - size] : ~r.first, earlier = begin > size ? keys[begin - size - 1] : ~r.first;
  const unsigned next_last = keys[next - 1], next_behind = next < n ? keys[next] : ~r.last;
  r.entered = before == r.first;
  const bool whole = r.entered && r.last == r.first;
  r.skip = r.entered && !(r.last == r.first && behind == r.first) && !(previous == r.first && earlier == r.first);
  const bool goes_on = behind == r.last && !whole, ends_next = !(next_last == r.last && next_behind == r.last);
  r.extended = goes_on && ends_next;
  r.leaves = goes_on && !ends_next;
  r.stop = r.extended ? next : r.end;
  return r;
}

// The chunks in which long runs begin: those of up to MANY_PARTS parts from the front of the list, the others from its back.
constexpr unsigned MANY_PARTS = 32;
struct long_runs { unsigned few, many, pad[62], chunks[1]; };

// the sum becomes a row of the result, added to what is there (`old`) if that is wanted
template <class O, int V, bool ADD> __device__ __forceinline__ void write_sum(O* to, const float (&sum)[V], float scale, const words<O, V>& old) {
  float f[V];
  if (ADD) channels(old, f);
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = ADD ? fmaf(sum[v], scale, f[v]) : sum[v] * scale;
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

// (keys, positions, partial and list are written by the kernels before this one and the join, while they may already be resident: not __restrict__, which would
// allow loads that are for data that does not change.)
template <class T, class O, int V, bool ADD>
__global__ void __launch_bounds__(GRAD_BLOCK, ADD ? 2 : 3) embedding_grad_kernel(const T* __restrict__ dout, size_t stride, const unsigned* keys, const unsigned* positions,
                                                                  size_t n, unsigned rows, unsigned pieces, grad_shape shape, float scale, unsigned zero_blocks,
                                                                  O* __restrict__ out, float* __restrict__ partial, long_runs* __restrict__ list, const tb200::ws_header* hdr) {
  tb200::grid_dependency_wait();        // the places are sorted
  tb200::grid_dependents_launch();      // the join may take its place
  const size_t dim = (size_t)pieces * V;
  if (hdr->error) {      // the sort's waits ran out
    for (size_t i = (size_t)blockIdx.x * GRAD_BLOCK + threadIdx.x; i < rows * dim; i += (size_t)gridDim.x * GRAD_BLOCK) out[i] = from_f32<O>(__int_as_float(0x7fffffff));
    return;
  }
  const unsigned sum_blocks = gridDim.x - zero_blocks;
  if (blockIdx.x >= sum_blocks) {      // behind the sums, which take longer
    __shared__ unsigned present;
    const unsigned first = (blockIdx.x - sum_blocks) * GRAD_ZERO, count = rows - first < GRAD_ZERO ? rows - first : GRAD_ZERO;
    if (threadIdx.x < 32) {      // a lane a row: is there a place of its token among those of the rows?  (Walking them takes as long as a frequent token has places.)
      const size_t from = warp_lower_bound(keys, n, first), to = warp_lower_bound(keys, n, first + count);
      size_t lo = from, hi = to;
      while (lo < hi) { const size_t mid = (lo + hi) >> 1; if (keys[mid] < first + threadIdx.x) lo = mid + 1; else hi = mid; }
      const unsigned all = __ballot_sync(tb200::FULL_MASK, threadIdx.x < count && lo < to && keys[lo] == first + threadIdx.x);
      if (threadIdx.x == 0) present = all;
    }
    __syncthreads();
    if constexpr (V > 1) {
      float none[V];
#pragma unroll
      for (int v = 0; v < V; ++v) none[v] = 0.f;
      for (unsigned r = 0; r < count; ++r)
        if (!(present >> r & 1))
          for (unsigned c = threadIdx.x; c < pieces; c += GRAD_BLOCK) store_words<O, V>(out + (size_t)(first + r) * dim + (size_t)c * V, to_words<O, V>(none));
    } else {      // of rows of any width neighbouring ones are one stretch of memory
      for (unsigned r = 0; r < count;) {
        if (present >> r & 1) { ++r; continue; }
        const unsigned from = r;
        while (r < count && !(present >> r & 1)) ++r;
        clear_stretch(out + (size_t)(first + from) * dim, out + (size_t)(first + r) * dim);
      }
    }
    return;
  }
  const share mine = share_of((size_t)blockIdx.x * GRAD_BLOCK + threadIdx.x, shape.spread, shape.parts);
  const size_t chunk = mine.at;
  const unsigned c = (mine.part << shape.spread) + mine.in;
  // What there is to do, place by place, found once for all columns: the row of dout to add (NO_ROW: none), and what becomes of the sum behind it: 0
  // nothing, 1 and 2 it is this chunk's part of a run that has begun earlier or goes on, 3 + v it is row v of the result.
  constexpr unsigned MOST = 2 * GRAD_CHUNK, NO_ROW = ~0u;
  __shared__ unsigned staged_keys[GRAD_BLOCK >> GRAD_SPREAD][MOST + 1];
  __shared__ __align__(16) unsigned staged_rows[GRAD_BLOCK >> GRAD_SPREAD][MOST], staged_then[GRAD_BLOCK >> GRAD_SPREAD][MOST];
  __shared__ unsigned staged_count[GRAD_BLOCK >> GRAD_SPREAD];
  const unsigned group = threadIdx.x >> shape.spread, step = 1u << shape.spread;
  unsigned* const its_keys = staged_keys[group];
  unsigned* const its_rows = staged_rows[group];
  unsigned* const its_then = staged_then[group];
  const size_t begin = chunk * shape.chunk;
  run_ends run = {};
  if (chunk < shape.chunks) {
    for (unsigned j = mine.in; j <= MOST; j += step) {
      const bool there = j <= 2 * shape.chunk && begin + j < n;
      its_keys[j] = there ? keys[begin + j] : ~0u;
      if (j < MOST) {
        const unsigned row = there ? positions[begin + j] : NO_ROW;
        its_rows[j] = row < n ? row : NO_ROW;
      }
    }
    run = run_ends_of(keys, n, chunk, shape.chunk);
    if (run.leaves && run.last < rows && mine.part == 0 && mine.in == 0) {
      const size_t far = (chunk + MANY_PARTS) * shape.chunk;      // a place of the part behind so many
      if (far < n && keys[far] == run.last) list->chunks[shape.chunks - 1 - atomicAdd(&list->many, 1u)] = (unsigned)chunk;
      else list->chunks[atomicAdd(&list->few, 1u)] = (unsigned)chunk;
    }
  }
  __syncthreads();
  if (chunk < shape.chunks) {
    const unsigned end = (unsigned)(run.end - begin), stop = (unsigned)(run.stop - begin);
    for (unsigned j = mine.in; j < MOST; j += step) {
      const unsigned key = its_keys[j];
      const bool here = j < end || (j < stop && key == run.last), used = here && key < rows && !(run.skip && key == run.first);
      const bool ends = its_keys[j + 1] != key, leaves = !ends && j + 1 == end && !run.extended;
      if (!used) its_rows[j] = NO_ROW;
      its_then[j] = !used || !(ends || leaves) ? 0u : run.entered && key == run.first ? 1u : leaves ? 2u : 3u + key;
      if (here && (j + 1 == MOST || !(j + 1 < end || (j + 1 < stop && its_keys[j + 1] == run.last)))) staged_count[group] = j + 1;
    }
  }
  __syncthreads();
  if (chunk >= shape.chunks || c >= pieces) return;
  const T* const from = dout + (size_t)c * V;
  const unsigned count = staged_count[group];
  float sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) sum[v] = 0.f;
  for (unsigned j0 = 0; j0 < count; j0 += GRAD_U) {
    words<T, V> r[GRAD_U] = {};
    words<O, V> old[GRAD_U];
    unsigned then[GRAD_U];
#pragma unroll
    for (int u = 0; u < GRAD_U; u += 4) {
      const uint4 at = *reinterpret_cast<const uint4*>(its_rows + j0 + u), th = *reinterpret_cast<const uint4*>(its_then + j0 + u);
      const unsigned row[4] = {at.x, at.y, at.z, at.w};
      then[u] = th.x; then[u + 1] = th.y; then[u + 2] = th.z; then[u + 3] = th.w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (row[i] != NO_ROW) r[u + i] = load_words<T, V>(from + (size_t)row[i] * stride);
        if (ADD && then[u + i] > 2) old[u + i] = load_words<O, V>(out + (size_t)(then[u + i] - 3) * dim + (size_t)c * V);
      }
    }
#pragma unroll
    for (int u = 0; u < GRAD_U; ++u) {
      float f[V];
      channels(r[u], f);
#pragma unroll
      for (int v = 0; v < V; ++v) sum[v] += f[v];
      if (then[u]) {
        if (then[u] > 2) write_sum<O, V, ADD>(out + (size_t)(then[u] - 3) * dim + (size_t)c * V, sum, scale, old[u]);
        else write_part<V>(partial + (2 * chunk + then[u] - 1) * dim + (size_t)c * V, sum);
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] = 0.f;
      }
    }
  }
}

// Runs of few parts: a warp takes one, 32 pieces of the columns at a time.  Of the others a CTA's eight warps add up neighbouring parts each, and their sums
// are added up in order.  (The order of the list is any; each run is by itself.)  About 10 us of those 163, mostly the way to the first part and back.
constexpr unsigned JOIN_WARPS = GRAD_BLOCK / 32;
template <class O, int V, bool ADD>
__global__ void __launch_bounds__(GRAD_BLOCK) embedding_grad_join_kernel(const unsigned* keys, unsigned pieces, grad_shape shape, float scale, O* __restrict__ out,
                                                                       const float* partial, const long_runs* list, const tb200::ws_header* hdr) {
  __shared__ size_t behind;            // the first chunk that has no part
  __shared__ float sums[JOIN_WARPS][32][V];
  tb200::grid_dependency_wait();
  if (hdr->error) return;
  constexpr int AHEAD = 8;
  const size_t dim = (size_t)pieces * V;
  const unsigned columns = (pieces + 31) / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32, few = list->few, many = list->many;
  for (unsigned long long item = (unsigned long long)blockIdx.x * JOIN_WARPS + warp; item < (unsigned long long)few * columns; item += (unsigned long long)gridDim.x * JOIN_WARPS) {
    const unsigned nth = (unsigned)(item / columns), c = (unsigned)(item - (unsigned long long)nth * columns) * 32 + lane;
    const size_t chunk = list->chunks[nth];
    const unsigned key = keys[(chunk + 1) * shape.chunk];
    const bool its = chunk + 1 + lane < shape.chunks && keys[(chunk + 1 + lane) * shape.chunk] == key;
    const unsigned parts = 1 + __popc(__ballot_sync(tb200::FULL_MASK, its));
    if (c < pieces) {
      const float* const p = partial + 2 * chunk * dim + (size_t)c * V;
      O* const at = out + (size_t)key * dim + (size_t)c * V;
      words<O, V> old;
      if (ADD) old = load_words<O, V>(at);
      float sum[V];
#pragma unroll
      for (int v = 0; v < V; ++v) sum[v] = 0.f;
      for (unsigned i = 0; i < parts; i += AHEAD) {
        float f[AHEAD][V];
#pragma unroll
        for (unsigned u = 0; u < AHEAD; ++u)
          if (i + u < parts) read_part<V>(p + (i + u ? 2 * (size_t)(i + u) : 1) * dim, f[u]);
#pragma unroll
        for (unsigned u = 0; u < AHEAD; ++u)
          if (i + u < parts) {
#pragma unroll
            for (int v = 0; v < V; ++v) sum[v] += f[u][v];
          }
      }
      write_sum<O, V, ADD>(at, sum, scale, old);
    }
  }
  for (unsigned long long item = blockIdx.x; item < (unsigned long long)many * columns; item += gridDim.x) {
    const unsigned nth = (unsigned)(item / columns), c = (unsigned)(item - (unsigned long long)nth * columns) * 32 + lane;
    const size_t chunk = list->chunks[shape.chunks - 1 - nth];
    const unsigned key = keys[(chunk + 1) * shape.chunk];
    if (warp == 0) {
      size_t q = chunk + 1;
      for (unsigned full = ~0u; full == ~0u; q += __popc(full)) full = __ballot_sync(tb200::FULL_MASK, q + lane < shape.chunks && keys[(q + lane) * shape.chunk] == key);
      if (lane == 0) behind = q;
    }
    __syncthreads();
    // parts 0, 1, ...: the second row of this chunk, the first rows of those behind it
    const size_t parts = behind - chunk, share = (parts + JOIN_WARPS - 1) / JOIN_WARPS, from = warp * share, to = from + share < parts ? from + share : parts;
    float sum[V];
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = 0.f;
    if (c < pieces) {
      const float* const p = partial + 2 * chunk * dim + (size_t)c * V;
      for (size_t i = from; i < to; i += AHEAD) {
        float f[AHEAD][V];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
          if (i + u < to) read_part<V>(p + (i + u ? 2 * (i + u) : 1) * dim, f[u]);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
          if (i + u < to) {
#pragma unroll
            for (int v = 0; v < V; ++v) sum[v] += f[u][v];
          }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) sums[warp][lane][v] = sum[v];
    __syncthreads();
    if (warp == 0 && c < pieces) {
      O* const at = out + (size_t)key * dim + (size_t)c * V;
      words<O, V> old;
      if (ADD) old = load_words<O, V>(at);
      for (unsigned w = 1; w < JOIN_WARPS && w * share < parts; ++w)
#pragma unroll
        for (int v = 0; v < V; ++v) sum[v] += sums[w][lane][v];
      write_sum<O, V, ADD>(at, sum, scale, old);
    }
    __syncthreads();
  }
}

// Chunks of GRAD_CHUNK places, smaller ones (down to 8) while fewer than a thousand threads a SM would have work.
constexpr size_t GRAD_THREADS = 148 * 1024;
grad_shape grad_shape_of(size_t n, size_t pieces) {
  grad_shape s;
  s.spread = spread_of(pieces, 8) < GRAD_SPREAD ? GRAD_SPREAD : spread_of(pieces, 8);
  s.parts = (unsigned)((pieces + (size_t(1) << s.spread) - 1) >> s.spread);
  s.chunk = GRAD_CHUNK;
  while (s.chunk > 8 && ((n + s.chunk - 1) / s.chunk * s.parts << s.spread) < GRAD_THREADS) s.chunk /= 2;
  s.chunks = (n + s.chunk - 1) / s.chunk;
  return s;
}

// the workspace: the sort's, then keys, positions and the sort's other halves, then the chunks' sums
struct grad_layout {
  size_t array, sort, list, partial, need;
  grad_layout(size_t n, size_t dim) {
    array = tb200::align_up(n * 4, 256);
    sort = tb200::align_up(tb200::radix_workspace_bytes<4, 4>(n), 256);
    // as many chunks as there can be, whatever the pieces: of 8 places, or GRAD_CHUNK and, where they are smaller, at most GRAD_THREADS to the half of them
    const grad_shape s = grad_shape_of(n, (dim + 7) / 8);
    const size_t most = n / GRAD_CHUNK + 2 * GRAD_THREADS / ((size_t)s.parts << s.spread) + 2, chunks = (n + 7) / 8 < most ? (n + 7) / 8 : most;
    list = sort + 4 * array;
    partial = list + tb200::align_up(256 + chunks * 4, 256);
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
        constexpr int LOOKUP_U = lookup_u(V, sizeof(T));
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
        const grad_layout lay(n, dim ? dim : 1);      // (no channels: nothing is done below, but the size may be asked for)
        int rc;
        if (workspace_gate(d_ws, ws_bytes, lay.need, rc)) return rc;
        if (rows == 0 || dim == 0) return 0;
        if (!d_out || (n && (!d_dout || !d_tokens)) || dout_stride < dim || dim >= (1ull << 31)) return ERR_INVALID;
        char* const base = static_cast<char*>(d_ws);
        unsigned* const keys = reinterpret_cast<unsigned*>(base + lay.sort);
        unsigned* const positions = reinterpret_cast<unsigned*>(base + lay.sort + 2 * lay.array);
        float* const partial = reinterpret_cast<float*>(base + lay.partial);
        long_runs* const list = reinterpret_cast<long_runs*>(base + lay.list);
        cudaError_t e;
        if (n && n <= PLACE_MOST) {
          auto place = [&](auto pv) {
            constexpr int P = decltype(pv)::value;
            place_kernel<P, I><<<(unsigned)((n + 32 * P - 1) / (32 * P)), PLACE_BLOCK, 0, stream>>>(static_cast<const I*>(d_tokens), (unsigned)n, (unsigned)rows, keys, positions, &list->few,
                                                                                                  static_cast<tb200::ws_header*>(d_ws));
          };
          if (n <= 32u * (unsigned)tb200::current_device_info().sm_count) place(std::integral_constant<int, 1>());
          else place(std::integral_constant<int, 2>());
          e = cudaGetLastError();
        } else {
          if (n) token_keys_kernel<I><<<(unsigned)((n + 255) / 256), 256, 0, stream>>>(static_cast<const I*>(d_tokens), n, (unsigned)rows, keys, positions, &list->few);
          tb200::key_coding coding;
          coding.kind = tb200::KEY_UNSIGNED;
          coding.descending = 0;
          int bits = 8;
          while (bits < 32 && (rows >> bits)) bits += 8;      // the largest key is `rows`
          // The sums below look for the sort's status in the header, so this sort reports there, announced or not.
          const void* const watched = tb200::thread_report().ws;
          tb200::thread_report().ws = nullptr;
          e = tb200::radix_sort_async<uint32_t, uint32_t, true>(keys, keys + lay.array / 4, positions, positions + lay.array / 4, n, coding, 0, bits, d_ws, stream);
          tb200::thread_report().ws = watched;
        }
        if (e != cudaSuccess) return (int)e;
        auto go = [&](auto vv, auto av) -> int {
          constexpr int V = decltype(vv)::value, JOIN_V = V < 4 ? V : 4;
          constexpr bool ADD = decltype(av)::value;
          const unsigned pieces = (unsigned)(dim / V), join_pieces = (unsigned)(dim / JOIN_V);
          const grad_shape shape = grad_shape_of(n, pieces);
          const tb200::ws_header* hdr = static_cast<const tb200::ws_header*>(d_ws);
          const unsigned zero_blocks = ADD ? 0u : (unsigned)((rows + GRAD_ZERO - 1) / GRAD_ZERO);
          const size_t grid = ((shape.chunks * shape.parts << shape.spread) + GRAD_BLOCK - 1) / GRAD_BLOCK;
          if (grid + zero_blocks > 0x7fffffffull) return ERR_INVALID;
          if (grid + zero_blocks == 0) return 0;
          const cudaError_t e = tb200::launch_after(embedding_grad_kernel<T, O, V, ADD>, grid + zero_blocks, GRAD_BLOCK, 0, stream, static_cast<const T*>(d_dout), dout_stride, keys, positions, n,
                                                    (unsigned)rows, pieces, shape, scale, zero_blocks, static_cast<O*>(d_out), partial, list, hdr);
          if (e != cudaSuccess || shape.chunks < 3) return (int)e;
          const size_t items = (join_pieces + 31) / 32 * shape.chunks / 2, most = (size_t)tb200::current_device_info().sm_count * 3;
          return (int)tb200::launch_after(embedding_grad_join_kernel<O, JOIN_V, ADD>, items < most ? items : most, GRAD_BLOCK, 0, stream, keys, join_pieces, shape, scale,
                                          static_cast<O*>(d_out), partial, list, hdr);
        };
        auto with = [&](auto vv) -> int { return accumulate ? go(vv, std::true_type()) : go(vv, std::false_type()); };
        // pieces of 16 bytes of the wider of the two types, at most 8 channels: both sides are aligned to theirs then
        constexpr int WIDE = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
        if (in_16_bytes(d_dout, dim, dout_stride, sizeof(T)) && in_16_bytes(d_out, dim, dim, sizeof(O))) return with(std::integral_constant<int, WIDE>());
        return with(std::integral_constant<int, 1>());
      });
    });
  });
}
