// C ABI: tb200_gated_scan, tb200_gated_scan_grad and tb200_gated_step.
#include "abi_rows.cuh"

using namespace tb200_abi;
using namespace tb200_rows;

namespace {
constexpr int BLOCK = 128;

// keep = 1 / (1 + exp(-g)) and give = 1 - keep, each to a few units in its last place: from e = exp(-|g|), which cannot overflow, so
// that the smaller of the two is e / (1 + e) and no difference of nearly equal numbers.
struct gate_pair { float keep, give; };
__device__ __forceinline__ gate_pair open_gate(float g) {
  const float e = __expf(-fabsf(g)), r = __fdividef(1.f, 1.f + e), s = e * r;
  gate_pair p;
  p.keep = g >= 0.f ? r : s;
  p.give = g >= 0.f ? s : r;
  return p;
}

// Where the sequences lie: from offsets if there are any, else `batch` of equal length.  Offsets that point outside are cut off.
template <class I> struct sequences {
  const I* offsets;
  size_t batch, n, length;
  __device__ size_t begin(size_t s) const {
    if (!offsets) return s * length;
    const long long o = (long long)offsets[s];
    return o < 0 ? 0 : (size_t)o > n ? n : (size_t)o;
  }
  __device__ size_t end(size_t s) const { return begin(s + 1); }
};

// a thread a channel of a sequence; the CTAs behind the last sequence's clear the rows that are in none
template <class T, class I>
__global__ void __launch_bounds__(BLOCK) gated_scan_kernel(const T* x, size_t xs, const T* gate, size_t gs, const float* h0, sequences<I> seq, size_t dim, T* h, float* last) {
  const size_t c = (size_t)blockIdx.y * BLOCK + threadIdx.x, s = blockIdx.x;
  if (c >= dim) return;
  if (s == seq.batch) {
    const size_t first = seq.begin(0), stop = seq.begin(seq.batch);
    for (size_t r = 0; r < first; ++r) h[r * dim + c] = from_f32<T>(0.f);
    for (size_t r = stop; r < seq.n; ++r) h[r * dim + c] = from_f32<T>(0.f);
    return;
  }
  float state = h0 ? h0[s * dim + c] : 0.f;
  const size_t end = seq.end(s);
  for (size_t r = seq.begin(s); r < end; ++r) {
    const gate_pair p = open_gate(to_f32(gate[r * gs + c]));
    state = p.keep * state + p.give * to_f32(x[r * xs + c]);
    h[r * dim + c] = from_f32<T>(state);
  }
  last[s * dim + c] = state;
}

template <class T, class I>
__global__ void __launch_bounds__(BLOCK) gated_scan_grad_kernel(const T* dh, size_t ds, const T* x, size_t xs, const T* gate, size_t gs, const T* h, size_t hs, const float* h0,
                                                              const float* dlast, sequences<I> seq, size_t dim, T* dx, T* dgate, float* dh0) {
  const size_t c = (size_t)blockIdx.y * BLOCK + threadIdx.x, s = blockIdx.x;
  if (c >= dim) return;
  if (s == seq.batch) {
    const size_t first = seq.begin(0), stop = seq.begin(seq.batch);
    for (size_t r = 0; r < seq.n; ++r)
      if (r < first || r >= stop) dx[r * dim + c] = dgate[r * dim + c] = from_f32<T>(0.f);
    return;
  }
  float carry = dlast ? dlast[s * dim + c] : 0.f;
  const size_t begin = seq.begin(s);
  for (size_t r = seq.end(s); r-- > begin;) {
    const gate_pair p = open_gate(to_f32(gate[r * gs + c]));
    const float total = to_f32(dh[r * ds + c]) + carry;
    const float before = r > begin ? to_f32(h[(r - 1) * hs + c]) : h0 ? h0[s * dim + c] : 0.f;
    dx[r * dim + c] = from_f32<T>(p.give * total);
    dgate[r * dim + c] = from_f32<T>(p.keep * p.give * (before - to_f32(x[r * xs + c])) * total);
    carry = p.keep * total;
  }
  dh0[s * dim + c] = carry;
}

// one token of each sequence: state[slot] is read and written, and is the row's output too
template <class T, class I>
__global__ void __launch_bounds__(BLOCK) gated_step_kernel(const T* x, size_t xs, const T* gate, size_t gs, float* state, size_t pool, const I* slots, size_t dim, T* h) {
  const size_t c = (size_t)blockIdx.y * BLOCK + threadIdx.x, r = blockIdx.x;
  if (c >= dim) return;
  const long long slot = slots ? (long long)slots[r] : (long long)r;
  float v = 0.f;
  if (slot >= 0 && (size_t)slot < pool) {
    const gate_pair p = open_gate(to_f32(gate[r * gs + c]));
    float* const at = state + (size_t)slot * dim + c;
    v = p.keep * *at + p.give * to_f32(x[r * xs + c]);
    *at = v;
  }
  h[r * dim + c] = from_f32<T>(v);
}

constexpr size_t MOST_CTAS_Y = 65535;
}  // namespace

TB200_API int tb200_gated_scan(const void* d_x, size_t x_stride, const void* d_gate, size_t gate_stride, const void* d_h0, const void* d_offsets, int offset_t, size_t batch,
                               size_t n, size_t dim, int t, void* d_h, void* d_last, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    return by_index_dtype(d_offsets ? offset_t : TB200_I32, [&](auto iv) -> int {
      using I = decltype(iv);
      if (dim == 0 || (n == 0 && batch == 0)) return 0;
      if ((n && (!d_x || !d_gate || !d_h)) || (batch && !d_last) || x_stride < dim || gate_stride < dim || batch >= 0x7fffffffull || (dim + BLOCK - 1) / BLOCK > MOST_CTAS_Y ||
          (!d_offsets && (batch == 0 || n % batch)))
        return ERR_INVALID;
      const sequences<I> seq = {static_cast<const I*>(d_offsets), batch, n, d_offsets ? 0 : n / batch};
      const dim3 grid((unsigned)(batch + (d_offsets ? 1 : 0)), (unsigned)((dim + BLOCK - 1) / BLOCK));
      gated_scan_kernel<T, I><<<grid, BLOCK, 0, stream>>>(static_cast<const T*>(d_x), x_stride, static_cast<const T*>(d_gate), gate_stride, static_cast<const float*>(d_h0), seq, dim,
                                                        static_cast<T*>(d_h), static_cast<float*>(d_last));
      return (int)cudaGetLastError();
    });
  });
}

TB200_API int tb200_gated_scan_grad(const void* d_dh, size_t dh_stride, const void* d_x, size_t x_stride, const void* d_gate, size_t gate_stride, const void* d_h, size_t h_stride,
                                    const void* d_h0, const void* d_dlast, const void* d_offsets, int offset_t, size_t batch, size_t n, size_t dim, int t, void* d_dx,
                                    void* d_dgate, void* d_dh0, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    return by_index_dtype(d_offsets ? offset_t : TB200_I32, [&](auto iv) -> int {
      using I = decltype(iv);
      if (dim == 0 || (n == 0 && batch == 0)) return 0;
      if ((n && (!d_dh || !d_x || !d_gate || !d_h || !d_dx || !d_dgate)) || (batch && !d_dh0) || dh_stride < dim || x_stride < dim || gate_stride < dim || h_stride < dim ||
          batch >= 0x7fffffffull || (dim + BLOCK - 1) / BLOCK > MOST_CTAS_Y || (!d_offsets && (batch == 0 || n % batch)))
        return ERR_INVALID;
      const sequences<I> seq = {static_cast<const I*>(d_offsets), batch, n, d_offsets ? 0 : n / batch};
      const dim3 grid((unsigned)(batch + (d_offsets ? 1 : 0)), (unsigned)((dim + BLOCK - 1) / BLOCK));
      gated_scan_grad_kernel<T, I><<<grid, BLOCK, 0, stream>>>(static_cast<const T*>(d_dh), dh_stride, static_cast<const T*>(d_x), x_stride, static_cast<const T*>(d_gate), gate_stride,
                                                             static_cast<const T*>(d_h), h_stride, static_cast<const float*>(d_h0), static_cast<const float*>(d_dlast), seq, dim,
                                                             static_cast<T*>(d_dx), static_cast<T*>(d_dgate), static_cast<float*>(d_dh0));
      return (int)cudaGetLastError();
    });
  });
}

TB200_API int tb200_gated_step(const void* d_x, size_t x_stride, const void* d_gate, size_t gate_stride, void* d_state, size_t pool, const void* d_slots, int slot_t, size_t n,
                               size_t dim, int t, void* d_h, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    return by_index_dtype(d_slots ? slot_t : TB200_I32, [&](auto iv) -> int {
      using I = decltype(iv);
      if (n == 0 || dim == 0) return 0;
      if (!d_x || !d_gate || !d_h || (pool && !d_state) || x_stride < dim || gate_stride < dim || n > 0x7fffffffull || (dim + BLOCK - 1) / BLOCK > MOST_CTAS_Y)
        return ERR_INVALID;
      const dim3 grid((unsigned)n, (unsigned)((dim + BLOCK - 1) / BLOCK));
      gated_step_kernel<T, I><<<grid, BLOCK, 0, stream>>>(static_cast<const T*>(d_x), x_stride, static_cast<const T*>(d_gate), gate_stride, static_cast<float*>(d_state), pool,
                                                        static_cast<const I*>(d_slots), dim, static_cast<T*>(d_h));
      return (int)cudaGetLastError();
    });
  });
}
