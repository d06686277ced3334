// C ABI: tb200_gated_scan, tb200_gated_scan_grad and tb200_gated_step.
#include <cuda.h>
#include <type_traits>

#include "abi_rows.cuh"
#include "thrust_b200/bulk_copy.cuh"

using namespace tb200_abi;
using namespace tb200_rows;

namespace {
constexpr int BLOCK = 128;

// keep = 1 / (1 + exp(-g)) and give = 1 - keep, from e = exp(-|g|), which cannot overflow, so that the smaller of the two is e / (1 + e) and no difference
// of nearly equal numbers.  The larger one is good to a few units in its last place, the smaller one to (8 + 1.2 |g|) of 2^-23: the exponential multiplies
// g by log2 e in 32 bits, and the fast exponential and reciprocal are what the scan's windows have time for (its gates are the longest part of a window).
struct gate_pair { float keep, give; };
__device__ __forceinline__ gate_pair open_gate(float g) {
  const float e = __expf(-fabsf(g)), r = __fdividef(1.f, 1.f + e), s = e * r;
  gate_pair p;
  p.keep = g >= 0.f ? r : s;
  p.give = g >= 0.f ? s : r;
  return p;
}

// ---------------------------------------------------------------------------------------------- scan by clusters
// A chain of rows (a sequence; packed sequences are one chain that is cut at their ends) is walked in windows by a cluster of CTAs, one
// chain and one slice of 64 channels each.  A lane has two neighbouring channels and ROWS neighbouring positions of a window in registers:
// position p is row p, or row length - 1 - p in the backward pass, so that both go the same way.  Over those positions a state q
// becomes A q + B in each channel.  The warps' pairs (A, B) meet in shared memory, the CTAs' in the shared memory of every CTA of the cluster, each
// thread folds what comes before its rows onto the carry of the window, and only then walks its rows again.  So each
// input is read once and each output written once.  Pairs are folded in the order of their positions: the same inputs give the same bits.
// States, pairs and sums are 32 bits; h, dx and dgate are rounded to the rows' type where they are stored, and nowhere before.
//
// A cut (a sequence begins there) makes a pair that forgets what came before: A is CUT instead of a product, and is selected on, not
// multiplied with, so that NaNs and infinities of one sequence do not reach the next.
//
// Where rows are made of whole 16-byte pieces, the copy engine brings a CTA's tiles (WARPS * ROWS rows of 64 channels of each input) into a
// ring of STAGES stages while earlier windows are worked on, and a lane takes its two channels of a row from there in one access.  Other rows (STAGES
// = 0) are read channel by channel where they are needed.  Two channels go through the arithmetic side by side (f32x2).
//
// What bounds it: with one CTA a chain the bytes (8 x 4096 bf16 rows of 2048: 82 us, 4910 GB/s; their gradient 143 us, 5620 GB/s, and 153 among other
// calls).  Where a cluster shares a chain, the length of a window: the gates about 860 cycles (two exponentials or reciprocals an element: the unit takes eight
// cycles for a warp's), the pairs' way through the warps 330, to the other CTAs and back 400, the rows 350, of which two CTAs a SM hide a part of one another's
// (one sequence of 20011 bf16 rows of 2560 76 us, its gradient 123, packed 101 and 165; of 65537 f32 rows of 1024 143 us).  Taking the next window's gates
// before this one's pairs have come needs twice the registers, and the CTA that has no room for them costs more than it saves (119 us and 196 when they took
// 71 and 171).  A chain has at most 16 CTAs for 64 channels: few channels leave SMs idle, however long the chain is.
constexpr float CUT = -1.f;

#ifdef TB200_TEST_HOOKS
// Test builds only (tests/cpp/gated_waits_test.cu, gated_waits_states_test.cu): the copies of window 1 of a cluster's first CTA are announced and not
// made; the pairs of window 1 of its last CTA are not sent.
__device__ unsigned withhold_copies, withhold_pairs;
__device__ __forceinline__ bool withheld(unsigned w, unsigned rank) { return withhold_copies && w == 1 && rank == 0; }
__device__ __forceinline__ bool pair_withheld(unsigned w, unsigned rank, unsigned ctas) { return withhold_pairs && w == 1 && rank == ctas - 1; }
#else
__device__ __forceinline__ bool withheld(unsigned, unsigned) { return false; }
__device__ __forceinline__ bool pair_withheld(unsigned, unsigned, unsigned) { return false; }
#endif

using f2 = unsigned long long;
__device__ __forceinline__ f2 pack2(float x, float y) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ float2 unpack2(f2 a) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { f2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 choose(bool c, f2 a, f2 b) { const float2 x = unpack2(a), y = unpack2(b); return pack2(c ? x.x : y.x, c ? x.y : y.y); }
__device__ __forceinline__ float exp2_of(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float one_over(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// two channels of a row, in a tile
template <class T> __device__ __forceinline__ float2 two_channels(const T* p) {
  const words<T, 2> w = load_words<T, 2>(p);
  return make_float2(channel<0>(w), channel<1>(w));
}

template <class T> struct rows_of { const T* at; size_t stride; };
// A lane's channels of up to ROWS rows, channel by channel.  Channels past the last are read as the last, rows that are not there as nothing in
// particular: no lane has a test of its own.
template <class T, int ROWS, bool EMPTY> struct direct_rows {
  T at[ROWS][2];
  __device__ __forceinline__ void request(const rows_of<T>& from, size_t row, int rows, int step, size_t c, size_t dim) {
    const size_t c0 = c < dim ? c : dim - 1;
    const unsigned next = c + 1 < dim ? 1 : 0;
    const T* q = from.at + row * from.stride + c0;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (i < rows) { at[i][0] = q[0]; at[i][1] = q[next]; }
      q = step > 0 ? q + from.stride : q - from.stride;
    }
  }
  __device__ __forceinline__ float2 get(int i) const { return make_float2(to_f32(at[i][0]), to_f32(at[i][1])); }
};
template <class T, int ROWS> struct direct_rows<T, ROWS, true> {};
// a lane's part of a row of states or of a result; PAIRS: both channels are there or none, and lie on a boundary of two
template <bool PAIRS> __device__ __forceinline__ f2 read_state(const float* p, bool first, bool second) {
  if constexpr (PAIRS) {
    if (!first) return 0ull;
    const float2 v = *reinterpret_cast<const float2*>(p);
    return pack2(v.x, v.y);
  } else {
    return pack2(first ? p[0] : 0.f, second ? p[1] : 0.f);
  }
}
template <bool PAIRS> __device__ __forceinline__ void write_state(float* p, float2 v, bool first, bool second) {
  if constexpr (PAIRS) {
    if (first) *reinterpret_cast<float2*>(p) = v;
  } else {
    if (first) p[0] = v.x;
    if (second) p[1] = v.y;
  }
}
template <bool PAIRS, class T> __device__ __forceinline__ void write_pair(T* p, const float (&v)[2], bool first, bool second) {
  if constexpr (PAIRS) {
    if (first) store_words<T, 2>(p, to_words<T, 2>(v));
  } else {
    if (first) p[0] = from_f32<T>(v[0]);
    if (second) p[1] = from_f32<T>(v[1]);
  }
}

// open_gate for two channels: e = exp(-g), keep = 1 / (1 + e), give = e keep.  From e = 2^25 on give is 1 to 32 bits and is not made from keep, which the
// reciprocal takes as zero where e is above 2^126; a NaN gate makes keep a NaN.
struct gates2 { f2 keep, give; };
__device__ __forceinline__ gates2 open_gates(float2 g) {
  constexpr float M = -1.4426950408889634f, ALL = 25.f;
  const float2 t = unpack2(mul2(pack2(g.x, g.y), pack2(M, M)));
  const f2 e = pack2(exp2_of(t.x), exp2_of(t.y));
  const float2 d = unpack2(add2(e, pack2(1.f, 1.f)));
  gates2 r;
  r.keep = pack2(one_over(d.x), one_over(d.y));
  const float2 give = unpack2(mul2(e, r.keep));
  r.give = pack2(t.x < ALL ? give.x : 1.f, t.y < ALL ? give.y : 1.f);
  return r;
}

struct duo { f2 a, b; };       // q becomes a q + b, in two channels
template <bool CUTS> __device__ __forceinline__ f2 follow(f2 q, duo f) {
  f2 r = fma2(f.a, q, f.b);
  if (CUTS) {
    const float2 a = unpack2(f.a), b = unpack2(f.b), s = unpack2(r);
    r = pack2(a.x == CUT ? b.x : s.x, a.y == CUT ? b.y : s.y);
  }
  return r;
}
// first f, then g
template <bool CUTS> __device__ __forceinline__ duo join(duo f, duo g) {
  duo r = {mul2(f.a, g.a), fma2(g.a, f.b, g.b)};
  if (CUTS) {
    const float2 fa = unpack2(f.a), ga = unpack2(g.a), gb = unpack2(g.b), a = unpack2(r.a), b = unpack2(r.b);
    r.a = pack2(fa.x == CUT || ga.x == CUT ? CUT : a.x, fa.y == CUT || ga.y == CUT ? CUT : a.y);
    r.b = pack2(ga.x == CUT ? gb.x : b.x, ga.y == CUT ? gb.y : b.y);
  }
  return r;
}

constexpr int MOST_CTAS = tb200::CLUSTER_MAX_CTAS;
constexpr int MEETINGS = 4;       // buffers of pairs; two are needed (join_ctas)
// Clusters of up to so many CTAs have room for no more pairs, and fold no more.  With room for 16 in all of them fewer clusters fit a SM's shared memory (20011 bf16
// rows: 60 slices get 9 CTAs each, 92 us and 168 with the gradient, or 6, 115 and 190; 150 slices 3, 242 and 455, or 2, 295 and 524; only the
// gradient of 100 slices, 5 or 4, is the faster for it, 274 against 295).  Larger clusters fold 16 either way.
constexpr unsigned FEW_CTAS = 9;
inline __host__ __device__ unsigned pair_slots(unsigned ctas) { return ctas > FEW_CTAS ? MOST_CTAS : FEW_CTAS; }
template <class T, int WARPS, int ROWS, int INPUTS, int STAGES> struct tiles_shared {
  static constexpr int R = WARPS * ROWS;
  static constexpr bool TILES = STAGES > 0;
  alignas(128) T tile[TILES ? STAGES : 1][TILES ? INPUTS : 1][TILES ? R : 1][64];
  duo warp[2][WARPS][32];
  unsigned long long full[TILES ? STAGES : 1], met[MEETINGS];
  // behind it, where there is more than one CTA: the CTAs' pairs, [MEETINGS][pair_slots][32]
  static size_t bytes(unsigned ctas) { return tb200::align_up(sizeof(tiles_shared), 16) + (ctas > 1 ? MEETINGS * pair_slots(ctas) * 32 * sizeof(duo) : 0); }
  __device__ duo* pairs() { return reinterpret_cast<duo*>(reinterpret_cast<char*>(this) + (sizeof(tiles_shared) + 15) / 16 * 16); }
};

__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* map, int channel, int row, unsigned long long* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(tb200::smem_addr(dst)), "l"(map), "r"(channel), "r"(row),
               "r"(tb200::smem_addr(bar)) : "memory");
}
// by whole warps; false: the copies did not come within the limit
__device__ __forceinline__ bool wait_tile(unsigned long long* bar, unsigned parity) {
  bool came = false;
  for (unsigned iter = 0; !came && iter < tb200::MBAR_SPIN_LIMIT; ++iter) came = tb200::mbar_try_wait(bar, parity);
  return __all_sync(tb200::FULL_MASK, came);
}
// a CTA that gives up: copies that were requested beyond the windows reached are not left in flight
template <int STAGES> __device__ __forceinline__ void wait_for_copies(unsigned long long* full, unsigned reached, unsigned tiles) {
  constexpr unsigned S = STAGES > 0 ? STAGES : 1;
  for (unsigned w = reached; w < tiles && w < reached + S; ++w) wait_tile(&full[w % S], w / S & 1);
}
// A 16-byte store into the shared memory of a CTA of the cluster, counted by the mbarrier there.  Unlike a barrier of the cluster it does not
// wait for this CTA's stores to global memory.
__device__ __forceinline__ void send_duo(unsigned to, const duo& d, unsigned bar) {
  const float2 a = unpack2(d.a), b = unpack2(d.b);
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "r"(bar) : "memory");
}
__device__ __forceinline__ bool wait_met(unsigned long long* bar, unsigned parity) {
  unsigned came = 0;
  for (unsigned iter = 0; !came && iter < tb200::MBAR_SPIN_LIMIT; ++iter)
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(came) : "r"(tb200::smem_addr(bar)), "r"(parity), "r"(1000u) : "memory");
  return __all_sync(tb200::FULL_MASK, came != 0);
}
__device__ __forceinline__ f2 nan2() { return pack2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff)); }

// where the shared memory of the CTAs lies that this warp sends to: one in WARPS (a single warp is a CTA that has no others)
template <int WARPS> struct peers { static constexpr int N = WARPS == 1 ? 1 : MOST_CTAS / WARPS; unsigned base[N]; };
struct link { duo before, total; };       // of the CTA: what comes before this warp's rows, all of it

// All threads of the CTA, with their warps' pairs of window w; `cut`: whether this warp's is one.  Behind it every warp is done with its tiles.
// Also sends the CTA's pair to the cluster.
template <class Shared, int WARPS, bool CUTS>
__device__ __forceinline__ link join_warps(Shared& sh, unsigned w, const duo& own, bool cut, unsigned rank, unsigned ctas, const peers<WARPS>& to, bool good) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  sh.warp[w & 1][warp][lane] = own;
  const bool some = CUTS ? __syncthreads_or(cut) != 0 : (__syncthreads(), false);
  link l;
  duo f = {pack2(1.f, 1.f), 0ull};
  l.before = f;
  if (CUTS && some) {
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      if (i == warp) l.before = f;
      f = join<true>(f, sh.warp[w & 1][i][lane]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      if (i == warp) l.before = f;
      f = join<false>(f, sh.warp[w & 1][i][lane]);
    }
  }
  l.total = f;
  if (ctas > 1) {
    const unsigned buffer = w % MEETINGS;
    if (threadIdx.x == 0 && good) tb200::mbar_arrive_expect(&sh.met[buffer], ctas * 32 * (unsigned)sizeof(duo));
    const unsigned base = tb200::smem_addr(&sh), at = tb200::smem_addr(sh.pairs() + (buffer * pair_slots(ctas) + rank) * 32 + lane) - base, bar = tb200::smem_addr(&sh.met[buffer]) - base;
#pragma unroll
    for (int k = 0; k < peers<WARPS>::N; ++k)
      if (warp + k * WARPS < (int)ctas && !pair_withheld(w, rank, ctas)) send_duo(to.base[k] + at, f, to.base[k] + bar);
  }
  return l;
}
// pairs that change nothing behind those of the cluster's CTAs
template <class Shared> __device__ __forceinline__ void no_pairs_behind(Shared& sh, unsigned ctas) {
  const unsigned slots = pair_slots(ctas), spare = (slots - ctas) * 32;
  const duo none = {pack2(1.f, 1.f), 0ull};
  for (unsigned i = threadIdx.x; i < MEETINGS * spare; i += blockDim.x) sh.pairs()[(i / spare * slots + ctas) * 32 + i % spare] = none;
}
// The state before this warp's rows of window w; `carry` goes from before the window to behind it.  false: the cluster's pairs did not come.
// A CTA sends window w + 1 when it has everything of w, which others sent when all their warps were done with w - 1: two buffers would do.
template <class Shared, bool CUTS>
__device__ __forceinline__ bool join_ctas(Shared& sh, unsigned w, const link& l, f2& carry, f2& q, unsigned rank, unsigned ctas, bool good) {
  if (ctas == 1) {
    q = follow<CUTS>(carry, l.before);
    carry = follow<CUTS>(carry, l.total);
    return true;
  }
  const bool met = good && wait_met(&sh.met[w % MEETINGS], w / MEETINGS & 1);
  // all steps the same, without a branch between them, so that the pairs are fetched together (behind the last CTA's there are pairs that change nothing):
  // nine steps with a test in each took 640 cycles of a window's 2900
  const duo* pairs = sh.pairs() + (w % MEETINGS) * pair_slots(ctas) * 32 + threadIdx.x % 32;
  f2 c = carry, here = carry;
  auto fold = [&](auto from, auto to) {
    constexpr unsigned FROM = decltype(from)::value, TO = decltype(to)::value;
    duo d[TO - FROM];
#pragma unroll
    for (unsigned r = FROM; r < TO; ++r) d[r - FROM] = pairs[r * 32];
#pragma unroll
    for (unsigned r = FROM; r < TO; ++r) {
      here = r == rank ? c : here;
      c = follow<CUTS>(c, d[r - FROM]);
    }
  };
  fold(std::integral_constant<unsigned, 0>(), std::integral_constant<unsigned, FEW_CTAS>());
  if (ctas > FEW_CTAS) fold(std::integral_constant<unsigned, FEW_CTAS>(), std::integral_constant<unsigned, MOST_CTAS>());
  q = follow<CUTS>(here, l.before);
  carry = c;
  return met;
}

// Which of the ROWS positions of a warp lie in a sequence, begin one and end one (in the direction of the walk), a bit each.  From a table with
// such bits for 32 rows an entry, read a window ahead.
struct marks { unsigned inside, begins, ends; };
struct row_table { const uint4* bits; const int* ids; };
// Of the rows from `row` on, a word a lane: lanes 0 to 2 the entry of the first of them, 4 to 6 the one behind it.
__device__ __forceinline__ unsigned read_marks(const row_table& t, long long row, long long length) {
  const int lane = threadIdx.x % 32;
  const long long k = (row >> 5) + (lane >> 2 & 1);
  return lane < 8 && k >= 0 && k <= (length - 1) >> 5 ? reinterpret_cast<const unsigned*>(t.bits + k)[lane & 3] : 0u;
}
template <int ROWS, bool BACKWARD> __device__ __forceinline__ marks marks_of(unsigned word, long long row) {
  auto cut_out = [&](int which) -> unsigned {
    const unsigned bits = __funnelshift_r(__shfl_sync(tb200::FULL_MASK, word, which), __shfl_sync(tb200::FULL_MASK, word, which + 4), (unsigned)row & 31);
    constexpr unsigned ALL = ROWS == 32 ? ~0u : (1u << (ROWS % 32)) - 1;
    return (BACKWARD ? __brev(bits) >> (32 - ROWS) : bits) & ALL;
  };
  marks m;
  m.inside = cut_out(0);
  m.begins = cut_out(BACKWARD ? 2 : 1);
  m.ends = cut_out(BACKWARD ? 1 : 2);
  return m;
}

template <class T, int WARPS, int ROWS, int STAGES, bool PACKED>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 1 ? 10 : STAGES == 0 ? 2 : PACKED ? 3 : 4)
gated_scan_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap gate_map, rows_of<T> x, rows_of<T> gate, const float* __restrict__ h0, row_table table, unsigned slices,
                   size_t length, size_t dim, T* __restrict__ h, float* __restrict__ last, tb200::ws_header* hdr) {
  static_assert(ROWS <= 32, "a lane holds the id of a position");
  using Shared = tiles_shared<T, WARPS, ROWS, 2, STAGES>;
  constexpr int R = Shared::R;
  constexpr unsigned ALL = ROWS == 32 ? ~0u : (1u << ROWS) - 1;
  extern __shared__ __align__(128) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const unsigned ctas = tb200::cluster_size(), rank = tb200::cluster_rank();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const unsigned item = blockIdx.x / ctas;
  const size_t chain = item / slices, c = (size_t)(item % slices) * 64 + lane * 2, first = chain * length;
  constexpr bool TILES = STAGES > 0;
  const bool there = c < dim, both = TILES ? there : c + 1 < dim;      // its channels
  const size_t window = (size_t)ctas * R;
  const unsigned windows = (unsigned)((length + window - 1) / window);
  const size_t p0 = ((size_t)rank * WARPS + warp) * ROWS;       // this warp's first position in window 0
  // the CTA has a tile in `tiles` windows
  const unsigned tiles = length > (size_t)rank * R ? (unsigned)((length - (size_t)rank * R + window - 1) / window) : 0;
  const int row0 = (int)(first + (size_t)rank * R), row_step = (int)window, channel0 = (int)(item % slices) * 64;
  auto load = [&](unsigned w) {
    if constexpr (!TILES) return;
    constexpr unsigned S = TILES ? STAGES : 1;
    if (w >= tiles) return;
    unsigned long long* const bar = &sh.full[w % S];
    const int row = row0 + (int)w * row_step;
    tb200::mbar_arrive_expect(bar, 2 * R * 64 * (unsigned)sizeof(T));
    if (withheld(w, rank)) return;
    load_tile(sh.tile[w % S][0], &x_map, channel0, row, bar);
    load_tile(sh.tile[w % S][1], &gate_map, channel0, row, bar);
  };
  if (threadIdx.x == 0) {
    if (blockIdx.x == 0) hdr->error = 0;      // a wait that runs out does so long after this
    for (int i = 0; i < STAGES; ++i) tb200::mbar_init(&sh.full[i], 1);
    for (int i = 0; i < MEETINGS; ++i) tb200::mbar_init(&sh.met[i], 1);
    tb200::mbar_init_fence();
    for (int i = 0; i < STAGES; ++i) load((unsigned)i);
  }
  auto state_of = [&](size_t s) -> f2 { return h0 ? read_state<TILES>(h0 + s * dim + c, there, both) : 0ull; };
  f2 carry = PACKED ? 0ull : state_of(chain);
  unsigned coming = 0;              // marks of the next window, and the ids of its rows, a lane a row
  int next_id = 0;
  auto id_at = [&](size_t p) -> int { return lane < ROWS && p + lane < length ? table.ids[p + lane] : 0; };
  if constexpr (PACKED) { coming = read_marks(table, (long long)p0, (long long)length); next_id = id_at(p0); }
  if (ctas > 1) no_pairs_behind(sh, ctas);
  __syncthreads();
  if (ctas > 1) tb200::cluster_barrier();      // all CTAs have begun: their shared memory may be written
  // Once a wait has run out nothing more is waited for, requested or announced; the results are NaNs from there on, and the kernel ends.
  bool good = true;
  unsigned reached = 0;        // windows whose tiles have come
  peers<WARPS> to;
#pragma unroll
  for (int k = 0; k < peers<WARPS>::N; ++k) to.base[k] = warp + k * WARPS < (int)ctas ? tb200::cluster_addr(tb200::smem_addr(&sh), warp + k * WARPS) : 0;

  struct held { f2 keep[ROWS], b[ROWS]; link l; unsigned cuts, ends; int id, rows; };
  auto take = [&](held& s, unsigned w) {
    const size_t p = p0 + w * window;
    constexpr unsigned S = TILES ? STAGES : 1;
    const unsigned stage = w % S;
    s.rows = p >= length ? 0 : length - p < (size_t)ROWS ? (int)(length - p) : ROWS;       // of this warp that there are
    s.cuts = s.ends = 0;
    unsigned begins = 0;
    f2 start = 0ull;
    if constexpr (PACKED) {
      const marks m = marks_of<ROWS, false>(coming, (long long)p);
      s.cuts = m.begins | (~m.inside & ALL);
      s.ends = m.ends;
      begins = m.begins;
      s.id = next_id;
      if (begins) start = state_of((size_t)__shfl_sync(tb200::FULL_MASK, s.id, __ffs(begins) - 1));      // on its way while the gates are worked out
      coming = read_marks(table, (long long)(p + window), (long long)length);
      next_id = id_at(p + window);
    }
    if (TILES && w < tiles && good) good = wait_tile(&sh.full[stage], w / S & 1);
    if (good) reached = w + 1;
    // the warp's rows of an input: in its tile, or all requested from where they lie
    direct_rows<T, ROWS, TILES> rx, rg;
    if constexpr (!TILES) {
      rx.request(x, first + p, s.rows, 1, c, dim);
      rg.request(gate, first + p, s.rows, 1, c, dim);
    }
    auto in = [&](int which, const direct_rows<T, ROWS, TILES>& from, int i) -> float2 {
      if constexpr (TILES) return two_channels(&sh.tile[stage][which][warp * ROWS + i][lane * 2]);
      else return from.get(i);
    };
    duo own = {pack2(1.f, 1.f), 0ull};
    auto open = [&](int i) {
      const gates2 g = open_gates(in(1, rg, i));
      const float2 xv = in(0, rx, i);
      s.keep[i] = g.keep;
      s.b[i] = mul2(g.give, pack2(xv.x, xv.y));
    };
    // Rows first, without a branch between them (their chains of exponential and reciprocal overlap: with a test in each row a window took 1.6 us
    // longer), then what is rare, then the pairs.
#pragma unroll
    for (int i = 0; i < ROWS; ++i) open(i);
    if (!PACKED && s.rows < ROWS) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (i >= s.rows) { s.keep[i] = pack2(1.f, 1.f); s.b[i] = 0ull; }
    }
    if (PACKED && s.cuts) {
      if (s.cuts == begins && (begins & (begins - 1)) == 0) {      // one beginning, as a rule: without a branch in each row
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
          s.b[i] = choose(begins >> i & 1, fma2(s.keep[i], start, s.b[i]), s.b[i]);
      } else {
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
          if (s.cuts >> i & 1) {
            if (begins >> i & 1) {
              if (begins & ((1u << i) - 1)) start = state_of((size_t)__shfl_sync(tb200::FULL_MASK, s.id, i));
              s.b[i] = fma2(s.keep[i], start, s.b[i]);
            } else {
              s.keep[i] = s.b[i] = 0ull;
            }
          }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) own.b = choose(s.cuts >> i & 1, s.b[i], fma2(s.keep[i], own.b, s.b[i]));
      own.a = pack2(CUT, CUT);
    } else {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        own.b = fma2(s.keep[i], own.b, s.b[i]);
        own.a = mul2(own.a, s.keep[i]);
      }
    }
    if (!good) own = {pack2(1.f, 1.f), nan2()};
    s.l = join_warps<Shared, WARPS, PACKED>(sh, w, own, s.cuts != 0, rank, ctas, to, good);
    if (threadIdx.x == 0 && good) load(w + STAGES);      // every warp has taken its rows from the tiles
  };
  auto give = [&](held& s, unsigned w) {
    f2 q = 0ull;
    good &= join_ctas<Shared, PACKED>(sh, w, s.l, carry, q, rank, ctas, good);
    if (!good) { q = carry = nan2(); s.cuts = 0; }      // what was folded may be anything
    T* hp = h + (first + p0 + w * window) * dim + c;
    if (s.rows == ROWS && !(PACKED && (s.cuts | s.ends))) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i, hp += dim) {
        q = fma2(s.keep[i], q, s.b[i]);
        const float2 v = unpack2(q);
        const float out[2] = {v.x, v.y};
        write_pair<TILES>(hp, out, there, both);
      }
    } else if (PACKED && s.rows == ROWS && (s.ends & (s.ends - 1)) == 0) {      // one end at most
      f2 end = 0ull;
#pragma unroll
      for (int i = 0; i < ROWS; ++i, hp += dim) {
        q = choose(s.cuts >> i & 1, s.b[i], fma2(s.keep[i], q, s.b[i]));
        end = choose(s.ends >> i & 1, q, end);
        const float2 v = unpack2(q);
        const float out[2] = {v.x, v.y};
        write_pair<TILES>(hp, out, there, both);
      }
      if (s.ends) {
        const int seq = __shfl_sync(tb200::FULL_MASK, s.id, __ffs(s.ends) - 1);
        write_state<TILES>(last + (size_t)seq * dim + c, unpack2(end), there, both);
      }
    } else {
#pragma unroll
      for (int i = 0; i < ROWS; ++i, hp += dim) {
        q = PACKED && (s.cuts >> i & 1) ? s.b[i] : fma2(s.keep[i], q, s.b[i]);
        const float2 v = unpack2(q);
        const float out[2] = {v.x, v.y};
        write_pair<TILES>(hp, out, there && i < s.rows, both && i < s.rows);
        if (PACKED && (s.ends >> i & 1)) {
          const int seq = __shfl_sync(tb200::FULL_MASK, s.id, i);
          write_state<TILES>(last + (size_t)seq * dim + c, v, there, both);
        }
      }
    }
  };
  held s;
  for (unsigned w = 0; w < windows; ++w) { take(s, w); give(s, w); }
  if (TILES && !good && warp == 0) wait_for_copies<STAGES>(sh.full, reached, tiles);
  if (ctas > 1) tb200::cluster_barrier();      // nobody leaves while something may still be sent there
  if (!good && lane == 0) tb200::record_error(&hdr->error, tb200::ERR_LOOKBACK_TIMEOUT);
  if (!PACKED && rank == 0 && warp == 0) write_state<TILES>(last + chain * dim + c, unpack2(carry), there, both);
}

template <class T, int WARPS, int ROWS, int STAGES, bool PACKED>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 1 ? 10 : STAGES == 0 ? 2 : PACKED ? 3 : 4)
gated_scan_grad_kernel(const __grid_constant__ CUtensorMap dh_map, const __grid_constant__ CUtensorMap gate_map, const __grid_constant__ CUtensorMap x_map,
                       const __grid_constant__ CUtensorMap h_map, rows_of<T> dh, rows_of<T> gate, rows_of<T> x, rows_of<T> h, const float* __restrict__ h0, const float* __restrict__ dlast, row_table table, unsigned slices,
                        size_t length, size_t dim, T* __restrict__ dx, T* __restrict__ dgate, float* __restrict__ dh0, tb200::ws_header* hdr) {
  static_assert(ROWS <= 32, "a lane holds the id of a position");
  using Shared = tiles_shared<T, WARPS, ROWS, 4, STAGES>;
  constexpr int R = Shared::R;
  constexpr unsigned ALL = ROWS == 32 ? ~0u : (1u << ROWS) - 1;
  extern __shared__ __align__(128) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const unsigned ctas = tb200::cluster_size(), rank = tb200::cluster_rank();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const unsigned item = blockIdx.x / ctas;
  const size_t chain = item / slices, c = (size_t)(item % slices) * 64 + lane * 2, first = chain * length;
  constexpr bool TILES = STAGES > 0;
  const bool there = c < dim, both = TILES ? there : c + 1 < dim;      // its channels
  const size_t window = (size_t)ctas * R;
  const unsigned windows = (unsigned)((length + window - 1) / window);
  const size_t p0 = ((size_t)rank * WARPS + warp) * ROWS;
  // the CTA has a tile in `tiles` windows; its position R - 1 is its first row, which may lie before the tensor
  const unsigned tiles = length > (size_t)rank * R ? (unsigned)((length - (size_t)rank * R + window - 1) / window) : 0;
  const int row0 = (int)((long long)first + (long long)length - (long long)rank * R - R), row_step = (int)window, channel0 = (int)(item % slices) * 64;
  auto load = [&](unsigned w) {
    if constexpr (!TILES) return;
    constexpr unsigned S = TILES ? STAGES : 1;
    if (w >= tiles) return;
    unsigned long long* const bar = &sh.full[w % S];
    const int row = row0 - (int)w * row_step;
    tb200::mbar_arrive_expect(bar, 4 * R * 64 * (unsigned)sizeof(T));
    if (withheld(w, rank)) return;
    load_tile(sh.tile[w % S][0], &dh_map, channel0, row, bar);
    load_tile(sh.tile[w % S][1], &gate_map, channel0, row, bar);
    load_tile(sh.tile[w % S][2], &x_map, channel0, row, bar);
    load_tile(sh.tile[w % S][3], &h_map, channel0, row - 1, bar);
  };
  if (threadIdx.x == 0) {
    if (blockIdx.x == 0) hdr->error = 0;      // a wait that runs out does so long after this
    for (int i = 0; i < STAGES; ++i) tb200::mbar_init(&sh.full[i], 1);
    for (int i = 0; i < MEETINGS; ++i) tb200::mbar_init(&sh.met[i], 1);
    tb200::mbar_init_fence();
    for (int i = 0; i < STAGES; ++i) load((unsigned)i);
  }
  auto state_of = [&](const float* from, size_t s) -> f2 { return from ? read_state<TILES>(from + s * dim + c, there, both) : 0ull; };
  f2 carry = PACKED ? 0ull : state_of(dlast, chain);
  const f2 initial = PACKED ? 0ull : state_of(h0, chain);
  unsigned coming = 0;
  int next_id = 0;
  auto id_at = [&](long long row) -> int { const long long at = row + ROWS - 1 - lane; return lane < ROWS && at >= 0 && at < (long long)length ? table.ids[at] : 0; };
  if constexpr (PACKED) {
    const long long row = (long long)length - (long long)p0 - ROWS;
    coming = read_marks(table, row, (long long)length);
    next_id = id_at(row);
  }
  if (ctas > 1) no_pairs_behind(sh, ctas);
  __syncthreads();
  if (ctas > 1) tb200::cluster_barrier();
  bool good = true;
  unsigned reached = 0;
  peers<WARPS> to;
#pragma unroll
  for (int k = 0; k < peers<WARPS>::N; ++k) to.base[k] = warp + k * WARPS < (int)ctas ? tb200::cluster_addr(tb200::smem_addr(&sh), warp + k * WARPS) : 0;

  struct held { f2 keep[ROWS], give[ROWS], d[ROWS], slope[ROWS]; link l; unsigned cuts, ends; int id, rows; };
  auto take = [&](held& s, unsigned w) {
    const size_t p = p0 + w * window;
    constexpr unsigned S = TILES ? STAGES : 1;
    const unsigned stage = w % S;
    s.rows = p >= length ? 0 : length - p < (size_t)ROWS ? (int)(length - p) : ROWS;
    s.cuts = s.ends = 0;
    unsigned begins = 0;
    f2 start = 0ull, from = initial;
    if constexpr (PACKED) {
      const long long row = (long long)length - (long long)p - ROWS;       // of the last position
      const marks m = marks_of<ROWS, true>(coming, row);
      s.cuts = m.begins | (~m.inside & ALL);
      s.ends = m.ends;
      begins = m.begins;
      s.id = next_id;
      if (begins) start = state_of(dlast, (size_t)__shfl_sync(tb200::FULL_MASK, s.id, __ffs(begins) - 1));
      if (s.ends) from = state_of(h0, (size_t)__shfl_sync(tb200::FULL_MASK, s.id, __ffs(s.ends) - 1));
      coming = read_marks(table, row - (long long)window, (long long)length);
      next_id = id_at(row - (long long)window);
    } else if (s.rows > 0 && p + s.rows == length) {
      s.ends = 1u << (s.rows - 1);           // the sequence's first row
    }
    if (TILES && w < tiles && good) good = wait_tile(&sh.full[stage], w / S & 1);
    if (good) reached = w + 1;
    direct_rows<T, ROWS, TILES> rd, rg, rx, rh;
    if constexpr (!TILES) {
      const size_t row = first + (length - 1 - (s.rows ? p : 0));
      rd.request(dh, row, s.rows, -1, c, dim);
      rg.request(gate, row, s.rows, -1, c, dim);
      rx.request(x, row, s.rows, -1, c, dim);
      rh.request(h, row - 1, s.rows - (s.rows > 0 && p + s.rows == length), -1, c, dim);      // the state before the chain's first row is not among them
    }
    auto in = [&](int which, const direct_rows<T, ROWS, TILES>& from, int i) -> float2 {
      if constexpr (TILES) return two_channels(&sh.tile[stage][which][R - 1 - warp * ROWS - i][lane * 2]);
      else return from.get(i);
    };
    const f2 minus = pack2(-1.f, -1.f);
    duo own = {pack2(1.f, 1.f), 0ull};
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const gates2 g = open_gates(in(1, rg, i));
      const float2 dv = in(0, rd, i), xv = in(2, rx, i), hv = in(3, rh, i);
      s.keep[i] = g.keep;
      s.give[i] = fma2(g.keep, 0ull, g.give);       // a NaN where the gate is one
      s.d[i] = pack2(dv.x, dv.y);
      s.slope[i] = mul2(mul2(g.keep, g.give), fma2(pack2(xv.x, xv.y), minus, pack2(hv.x, hv.y)));
    }
    if (s.ends && (s.ends & (s.ends - 1)) == 0) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const float2 xv = in(2, rx, i);
        s.slope[i] = choose(s.ends >> i & 1, mul2(mul2(s.keep[i], s.give[i]), fma2(pack2(xv.x, xv.y), minus, from)), s.slope[i]);
      }
    } else if (s.ends) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (s.ends >> i & 1) {
          if (s.ends & ((1u << i) - 1)) from = state_of(h0, (size_t)__shfl_sync(tb200::FULL_MASK, s.id, i));
          const float2 xv = in(2, rx, i);
          s.slope[i] = mul2(mul2(s.keep[i], s.give[i]), fma2(pack2(xv.x, xv.y), minus, from));
        }
    }
    if (!PACKED && s.rows < ROWS) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (i >= s.rows) { s.keep[i] = pack2(1.f, 1.f); s.give[i] = s.d[i] = s.slope[i] = 0ull; }
    }
    if (PACKED && s.cuts) {
      if (s.cuts == begins && (begins & (begins - 1)) == 0) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) s.d[i] = choose(begins >> i & 1, add2(s.d[i], start), s.d[i]);
      } else {
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
          if (s.cuts >> i & 1) {
            if (begins >> i & 1) {
              if (begins & ((1u << i) - 1)) start = state_of(dlast, (size_t)__shfl_sync(tb200::FULL_MASK, s.id, i));
              s.d[i] = add2(s.d[i], start);
            } else {
              s.keep[i] = s.give[i] = s.d[i] = s.slope[i] = 0ull;
            }
          }
      }
#pragma unroll
      for (int i = 0; i < ROWS; ++i) own.b = mul2(s.keep[i], choose(s.cuts >> i & 1, s.d[i], add2(own.b, s.d[i])));
      own.a = pack2(CUT, CUT);
    } else {
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        own.b = mul2(s.keep[i], add2(own.b, s.d[i]));
        own.a = mul2(own.a, s.keep[i]);
      }
    }
    if (!good) own = {pack2(1.f, 1.f), nan2()};
    s.l = join_warps<Shared, WARPS, PACKED>(sh, w, own, s.cuts != 0, rank, ctas, to, good);
    if (threadIdx.x == 0 && good) load(w + STAGES);      // every warp has taken its rows from the tiles
  };
  auto give = [&](held& s, unsigned w) {
    f2 q = 0ull;
    good &= join_ctas<Shared, PACKED>(sh, w, s.l, carry, q, rank, ctas, good);
    if (!good) { q = carry = nan2(); s.cuts = 0; }      // what was folded may be anything
    const long long at = ((long long)first + (long long)length - 1 - (long long)(p0 + w * window)) * (long long)dim + (long long)c;
    T* xp = dx + at;
    T* gp = dgate + at;
    if (s.rows == ROWS && !(PACKED && (s.cuts | s.ends))) {
#pragma unroll
      for (int i = 0; i < ROWS; ++i, xp -= dim, gp -= dim) {
        const f2 sum = add2(s.d[i], q);
        q = mul2(s.keep[i], sum);
        const float2 a = unpack2(mul2(s.give[i], sum)), b = unpack2(mul2(s.slope[i], sum));
        const float oa[2] = {a.x, a.y}, ob[2] = {b.x, b.y};
        write_pair<TILES>(xp, oa, there, both);
        write_pair<TILES>(gp, ob, there, both);
      }
    } else if (PACKED && s.rows == ROWS && (s.ends & (s.ends - 1)) == 0) {
      f2 end = 0ull;
#pragma unroll
      for (int i = 0; i < ROWS; ++i, xp -= dim, gp -= dim) {
        const f2 sum = choose(s.cuts >> i & 1, s.d[i], add2(s.d[i], q));
        q = mul2(s.keep[i], sum);
        end = choose(s.ends >> i & 1, q, end);
        const float2 a = unpack2(mul2(s.give[i], sum)), b = unpack2(mul2(s.slope[i], sum));
        const float oa[2] = {a.x, a.y}, ob[2] = {b.x, b.y};
        write_pair<TILES>(xp, oa, there, both);
        write_pair<TILES>(gp, ob, there, both);
      }
      if (s.ends) {
        const int seq = __shfl_sync(tb200::FULL_MASK, s.id, __ffs(s.ends) - 1);
        write_state<TILES>(dh0 + (size_t)seq * dim + c, unpack2(end), there, both);
      }
    } else {
#pragma unroll
      for (int i = 0; i < ROWS; ++i, xp -= dim, gp -= dim) {
        const f2 sum = PACKED && (s.cuts >> i & 1) ? s.d[i] : add2(s.d[i], q);
        q = mul2(s.keep[i], sum);
        const float2 a = unpack2(mul2(s.give[i], sum)), b = unpack2(mul2(s.slope[i], sum));
        const float oa[2] = {a.x, a.y}, ob[2] = {b.x, b.y};
        write_pair<TILES>(xp, oa, there && i < s.rows, both && i < s.rows);
        write_pair<TILES>(gp, ob, there && i < s.rows, both && i < s.rows);
        if (PACKED && (s.ends >> i & 1)) {
          const int seq = __shfl_sync(tb200::FULL_MASK, s.id, i);
          write_state<TILES>(dh0 + (size_t)seq * dim + c, unpack2(q), there, both);
        }
      }
    }
  };
  held s;
  for (unsigned w = 0; w < windows; ++w) { take(s, w); give(s, w); }
  if (TILES && !good && warp == 0) wait_for_copies<STAGES>(sh.full, reached, tiles);
  if (ctas > 1) tb200::cluster_barrier();
  if (!good && lane == 0) tb200::record_error(&hdr->error, tb200::ERR_LOOKBACK_TIMEOUT);
  if (!PACKED && rank == 0 && warp == 0) write_state<TILES>(dh0 + chain * dim + c, unpack2(carry), there, both);
}

// ids[r] = the sequence of row r, -1 if it is in none; bits[r / 32]: whether the rows are in one, begin one, end one.  A sequence without rows hands
// its state (or its gradient) on.
template <class I>
__global__ void __launch_bounds__(256) row_table_kernel(const I* offsets, size_t batch, size_t n, int* ids, uint4* bits, const float* from, size_t dim, float* to, tb200::ws_header* hdr) {
  if (blockIdx.x == 0 && threadIdx.x == 0) hdr->error = 0;
  const size_t r = (size_t)blockIdx.x * 256 + threadIdx.x;
  auto at = [&](size_t s) -> size_t { const long long o = (long long)offsets[s]; return o < 0 ? 0 : (size_t)o > n ? n : (size_t)o; };
  bool inside = false, begins = false, ends = false;
  if (r < n) {
    size_t lo = 0, hi = batch + 1;          // how many of the offsets are at most r
    while (lo < hi) { const size_t mid = (lo + hi) >> 1; if (at(mid) <= r) lo = mid + 1; else hi = mid; }
    inside = lo > 0 && lo <= batch;
    ids[r] = inside ? (int)(lo - 1) : -1;
    begins = inside && at(lo - 1) == r;
    ends = inside && at(lo) == r + 1;
  }
  const unsigned in = __ballot_sync(tb200::FULL_MASK, inside), first = __ballot_sync(tb200::FULL_MASK, begins), final = __ballot_sync(tb200::FULL_MASK, ends);
  if (threadIdx.x % 32 == 0 && r < n) bits[r / 32] = make_uint4(in, first, final, 0);
  for (size_t s = blockIdx.x; s < batch; s += gridDim.x)
    if (at(s) >= at(s + 1))
      for (size_t c = threadIdx.x; c < dim; c += 256) to[s * dim + c] = from ? from[s * dim + c] : 0.f;
}

// How many clusters of each size the device holds at once, for a kernel: asked once a kernel, device and host thread.
struct cluster_room { const void* kernel = nullptr; int device = -1; int clusters[MOST_CTAS + 1]; };
template <class... Params> const cluster_room& room_for(void (*kernel)(Params...), int block, size_t smem_few, size_t smem_most) {
  constexpr int KEPT = 32;
  static thread_local cluster_room kept[KEPT];
  static thread_local int next = 0;
  int device = 0;
  cudaGetDevice(&device);
  for (const cluster_room& r : kept) if (r.kernel == (const void*)kernel && r.device == device) return r;
  cluster_room& r = kept[next++ % KEPT];
  r.kernel = (const void*)kernel;
  r.device = device;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_most) != cudaSuccess ||
      cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    cudaGetLastError();
  for (int c = 2; c <= MOST_CTAS; ++c) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)c);
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = (unsigned)c > FEW_CTAS ? smem_most : smem_few;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)c; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&r.clusters[c], kernel, &cfg) != cudaSuccess) { cudaGetLastError(); r.clusters[c] = 0; }
  }
  return r;
}

// Whether the chains' slices fill the device by themselves: then one CTA walks a chain, and no pairs travel.  Sequences of 4096 bf16 rows of 2048, alone / shared:
// 192 slices 82 / 68 us (gradient 141 / 115), 224 slices 82 / 82 (143 / 138), 256 slices 82 / 84 (143 / 158), 320 slices 107 / 104 (201 / 184).
inline bool walked_alone(size_t chains, size_t dim) { return chains * ((dim + 63) / 64) >= 200; }

// Launches `kernel` on all chains and slices.  How many CTAs walk a chain together: as many as there are tiles, but no more than let all clusters run at
// once, since a second round costs more than any window saved (40 slices of 20011 bf16 rows: 10 CTAs 76 us, 9 76, 8 83, 7 91, and 11, of which not all fit, 109; 16
// slices of 65537 f32 rows: 13 CTAs 143, 12 152, 9 178, 14 229).
template <class Shared, class... Params, class... Args>
cudaError_t launch_chains(void (*kernel)(Params...), unsigned warps, bool alone, size_t chains, size_t length, size_t dim, cudaStream_t stream, Args... args) {
  const size_t items = chains * ((dim + 63) / 64), tiles = (length + Shared::R - 1) / Shared::R;
  unsigned ctas = 1;
  if (!alone && tiles > 1) {
    const cluster_room& room = room_for(kernel, (int)warps * 32, Shared::bytes(2), Shared::bytes(MOST_CTAS));
    ctas = tiles < (size_t)MOST_CTAS ? (unsigned)tiles : MOST_CTAS;
    while (ctas > 1 && (size_t)room.clusters[ctas] < items) --ctas;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = Shared::bytes(ctas);
  if (cfg.dynamicSmemBytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shared::bytes(MOST_CTAS));
    if (e != cudaSuccess) return e;
  }
  cfg.gridDim = dim3((unsigned)(items * ctas));
  cfg.blockDim = dim3(warps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
  if (ctas > 1 && tb200::launch_refused(e)) {      // no room for such a cluster after all: a CTA walks a chain alone
    cfg.gridDim = dim3((unsigned)items);
    attr[0].val.clusterDim.x = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
  }
  return e;
}

// One token of each sequence: state[slot] is read and written, and is the row's output too.  A thread has up to STEP_U pieces of V channels of a row; bound by the
// bytes of states and rows: 0.8 us of them for 96 bf16 rows of 4096, where the whole call takes 10.
constexpr int STEP_U = 2;
template <class T, int V, class I>
__global__ void __launch_bounds__(BLOCK) gated_step_kernel(const T* __restrict__ x, size_t xs, const T* __restrict__ gate, size_t gs, float* state, size_t pool, const I* __restrict__ slots,
                                                         size_t n, unsigned pieces, unsigned spread, unsigned parts, T* __restrict__ h) {
  const share s = share_of((size_t)blockIdx.x * BLOCK + threadIdx.x, spread, parts);
  const size_t r = s.at;
  if (r >= n) return;
  const unsigned lanes = 1u << spread, c0 = s.part * lanes * STEP_U + s.in;
  const long long slot = slots ? (long long)slots[r] : (long long)r;
  const bool there = slot >= 0 && (size_t)slot < pool;
  float* const at = state + (there ? (size_t)slot * pieces * V : 0);
  words<T, V> xw[STEP_U], gw[STEP_U];
  words<float, V> old[STEP_U];
#pragma unroll
  for (int u = 0; u < STEP_U; ++u) {
    const size_t c = (size_t)(c0 + u * lanes) * V;
    if (there && c0 + u * lanes < pieces) {
      xw[u] = load_words<T, V>(x + r * xs + c);
      gw[u] = load_words<T, V>(gate + r * gs + c);
      old[u] = load_words<float, V>(at + c);
    }
  }
#pragma unroll
  for (int u = 0; u < STEP_U; ++u) {
    if (c0 + u * lanes >= pieces) break;
    const size_t c = (size_t)(c0 + u * lanes) * V;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
    if (there) {
      float xv[V], gv[V];
      channels(xw[u], xv);
      channels(gw[u], gv);
      channels(old[u], v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const gate_pair p = open_gate(gv[i]);
        v[i] = fmaf(p.keep, v[i], p.give * xv[i]);
      }
      store_words<float, V>(at + c, to_words<float, V>(v));
    }
    store_words<T, V>(h + r * pieces * V + c, to_words<T, V>(v));
  }
}

// the workspace: header, then the rows' sequences where there are offsets
size_t scan_workspace(const void* offsets, size_t n) { return sizeof(tb200::ws_header) + (offsets ? tb200::align_up(n * 4, 256) + tb200::align_up((n + 31) / 32 * 16, 256) : 0); }
int* ids_of(void* d_ws) { return reinterpret_cast<int*>(static_cast<char*>(d_ws) + sizeof(tb200::ws_header)); }
uint4* bits_of(void* d_ws, size_t n) { return reinterpret_cast<uint4*>(static_cast<char*>(d_ws) + sizeof(tb200::ws_header) + tb200::align_up(n * 4, 256)); }

template <class I>
cudaError_t find_ids(const void* offsets, size_t batch, size_t n, void* d_ws, const void* from, size_t dim, void* to, cudaStream_t stream) {
  row_table_kernel<I><<<(unsigned)(n / 256 + 1), 256, 0, stream>>>(static_cast<const I*>(offsets), batch, n, ids_of(d_ws), bits_of(d_ws, n), static_cast<const float*>(from), dim, static_cast<float*>(to),
                                                               static_cast<tb200::ws_header*>(d_ws));
  return cudaGetLastError();
}

// The rows as the copy engine takes tiles of `box` rows of 64 channels from them; false: it cannot.
template <class T> bool tile_map(CUtensorMap& map, const void* p, size_t rows, size_t dim, size_t stride, unsigned box) {
  using encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const encode call = []() -> encode {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
    return reinterpret_cast<encode>(f);
  }();
  if (!in_16_bytes(p, dim, stride, sizeof(T)) || rows >= (1ull << 31) - 512) return false;
  const cuuint64_t dims[2] = {dim, rows}, strides[1] = {stride * sizeof(T)};
  const cuuint32_t boxes[2] = {64, box}, steps[2] = {1, 1};
  const CUtensorMapDataType type = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : std::is_same<T, f16>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  return call && call(&map, type, 2, const_cast<void*>(p), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Four warps of 16 rows (backward: of 8), one warp where a chain is no longer than 16.  Two stages leave room for four CTAs a SM; a CTA that walks a chain
// alone gains from a third (8 x 4096 bf16 rows of 2048: 82 us against 88, gradient 143 against 156; five: 83 and 148).
constexpr int SCAN_WARPS = 4, SCAN_ROWS = 16, GRAD_ROWS = 8, SHORT = 16;
using few_warps = std::integral_constant<int, SCAN_WARPS>;
using one_warp = std::integral_constant<int, 1>;
using no_stages = std::integral_constant<int, 0>;
using stages_shared = std::integral_constant<int, 2>;
using stages_alone = std::integral_constant<int, 3>;

bool scan_sizes_fit(const void* offsets, size_t batch, size_t n, size_t dim) {
  return batch < (1ull << 31) && n < (1ull << 40) && (offsets || (batch > 0 && n % batch == 0)) && n / 16 < (1ull << 31) - 1 && (offsets ? 1 : batch) * ((dim + 63) / 64) * MOST_CTAS < (1ull << 31) &&
         n / 256 < (1ull << 31) - 1;
}
}  // namespace

TB200_API int tb200_gated_scan(const void* d_x, size_t x_stride, const void* d_gate, size_t gate_stride, const void* d_h0, const void* d_offsets, int offset_t, size_t batch,
                               size_t n, size_t dim, int t, void* d_h, void* d_last, void* d_ws, size_t* ws_bytes, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    return by_index_dtype(d_offsets ? offset_t : TB200_I32, [&](auto iv) -> int {
      using I = decltype(iv);
      int rc;
      if (workspace_gate(d_ws, ws_bytes, scan_workspace(d_offsets, n), rc)) return rc;
      if (dim == 0 || (n == 0 && batch == 0)) return 0;
      if ((n && (!d_x || !d_gate || !d_h)) || (batch && !d_last) || x_stride < dim || gate_stride < dim || !scan_sizes_fit(d_offsets, batch, n, dim)) return ERR_INVALID;
      if (d_offsets) {
        const cudaError_t e = find_ids<I>(d_offsets, batch, n, d_ws, d_h0, dim, d_last, stream);
        if (e != cudaSuccess || n == 0) return (int)e;
      }
      const size_t chains = d_offsets ? 1 : batch, length = n / chains;
      const unsigned slices = (unsigned)((dim + 63) / 64);
      const bool alone = length <= SHORT || walked_alone(chains, dim);
      auto go = [&](auto warps, auto stages, const CUtensorMap& xm, const CUtensorMap& gm) -> int {
        constexpr int WARPS = decltype(warps)::value, STAGES = decltype(stages)::value;
        auto with = [&](auto packed) -> int {
          return (int)launch_chains<tiles_shared<T, WARPS, SCAN_ROWS, 2, STAGES>>(gated_scan_kernel<T, WARPS, SCAN_ROWS, STAGES, decltype(packed)::value>, WARPS, alone, chains, length, dim,
                                                                               stream, xm, gm, rows_of<T>{static_cast<const T*>(d_x), x_stride},
                                                                               rows_of<T>{static_cast<const T*>(d_gate), gate_stride}, static_cast<const float*>(d_h0),
                                                                               row_table{bits_of(d_ws, n), ids_of(d_ws)}, slices, length, dim, static_cast<T*>(d_h),
                                                                               static_cast<float*>(d_last), static_cast<tb200::ws_header*>(d_ws));
        };
        return d_offsets ? with(std::true_type()) : with(std::false_type());
      };
      CUtensorMap xm = {}, gm = {};
      constexpr unsigned BOX = SCAN_WARPS * SCAN_ROWS;
      if (length <= SHORT) return go(one_warp(), no_stages(), xm, gm);
      if (in_16_bytes(d_h, dim, dim, sizeof(T)) && in_16_bytes(d_h0, dim, dim, 4) && in_16_bytes(d_last, dim, dim, 4) && tile_map<T>(xm, d_x, n, dim, x_stride, BOX) &&
          tile_map<T>(gm, d_gate, n, dim, gate_stride, BOX))
        return alone ? go(few_warps(), stages_alone(), xm, gm) : go(few_warps(), stages_shared(), xm, gm);
      return go(few_warps(), no_stages(), xm, gm);
    });
  });
}

TB200_API int tb200_gated_scan_grad(const void* d_dh, size_t dh_stride, const void* d_x, size_t x_stride, const void* d_gate, size_t gate_stride, const void* d_h, size_t h_stride,
                                    const void* d_h0, const void* d_dlast, const void* d_offsets, int offset_t, size_t batch, size_t n, size_t dim, int t, void* d_dx,
                                    void* d_dgate, void* d_dh0, void* d_ws, size_t* ws_bytes, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    return by_index_dtype(d_offsets ? offset_t : TB200_I32, [&](auto iv) -> int {
      using I = decltype(iv);
      int rc;
      if (workspace_gate(d_ws, ws_bytes, scan_workspace(d_offsets, n), rc)) return rc;
      if (dim == 0 || (n == 0 && batch == 0)) return 0;
      if ((n && (!d_dh || !d_x || !d_gate || !d_h || !d_dx || !d_dgate)) || (batch && !d_dh0) || dh_stride < dim || x_stride < dim || gate_stride < dim || h_stride < dim ||
          !scan_sizes_fit(d_offsets, batch, n, dim))
        return ERR_INVALID;
      if (d_offsets) {
        const cudaError_t e = find_ids<I>(d_offsets, batch, n, d_ws, d_dlast, dim, d_dh0, stream);
        if (e != cudaSuccess || n == 0) return (int)e;
      }
      const size_t chains = d_offsets ? 1 : batch, length = n / chains;
      const unsigned slices = (unsigned)((dim + 63) / 64);
      const bool alone = length <= SHORT || walked_alone(chains, dim);
      auto go = [&](auto warps, auto stages, const CUtensorMap& dm, const CUtensorMap& gm, const CUtensorMap& xm, const CUtensorMap& hm) -> int {
        constexpr int WARPS = decltype(warps)::value, STAGES = decltype(stages)::value;
        auto with = [&](auto packed) -> int {
          return (int)launch_chains<tiles_shared<T, WARPS, GRAD_ROWS, 4, STAGES>>(
              gated_scan_grad_kernel<T, WARPS, GRAD_ROWS, STAGES, decltype(packed)::value>, WARPS, alone, chains, length, dim, stream, dm, gm, xm, hm,
              rows_of<T>{static_cast<const T*>(d_dh), dh_stride}, rows_of<T>{static_cast<const T*>(d_gate), gate_stride}, rows_of<T>{static_cast<const T*>(d_x), x_stride},
              rows_of<T>{static_cast<const T*>(d_h), h_stride}, static_cast<const float*>(d_h0), static_cast<const float*>(d_dlast), row_table{bits_of(d_ws, n), ids_of(d_ws)}, slices,
              length, dim, static_cast<T*>(d_dx), static_cast<T*>(d_dgate), static_cast<float*>(d_dh0), static_cast<tb200::ws_header*>(d_ws));
        };
        return d_offsets ? with(std::true_type()) : with(std::false_type());
      };
      CUtensorMap dm = {}, gm = {}, xm = {}, hm = {};
      constexpr unsigned BOX = SCAN_WARPS * GRAD_ROWS;
      if (length <= SHORT) return go(one_warp(), no_stages(), dm, gm, xm, hm);
      if (in_16_bytes(d_dx, dim, dim, sizeof(T)) && in_16_bytes(d_dgate, dim, dim, sizeof(T)) && in_16_bytes(d_h0, dim, dim, 4) && in_16_bytes(d_dlast, dim, dim, 4) &&
          in_16_bytes(d_dh0, dim, dim, 4) && tile_map<T>(dm, d_dh, n, dim, dh_stride, BOX) && tile_map<T>(gm, d_gate, n, dim, gate_stride, BOX) &&
          tile_map<T>(xm, d_x, n, dim, x_stride, BOX) && tile_map<T>(hm, d_h, n, dim, h_stride, BOX))
        return alone ? go(few_warps(), stages_alone(), dm, gm, xm, hm) : go(few_warps(), stages_shared(), dm, gm, xm, hm);
      return go(few_warps(), no_stages(), dm, gm, xm, hm);
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
      if (!d_x || !d_gate || !d_h || (pool && !d_state) || x_stride < dim || gate_stride < dim || n > 0x7fffffffull || dim >= (1ull << 31)) return ERR_INVALID;
      auto go = [&](auto vv) -> int {
        constexpr int V = decltype(vv)::value;
        const unsigned pieces = (unsigned)(dim / V), spread = spread_of((pieces + STEP_U - 1) / STEP_U, 5), parts = (unsigned)(((size_t)pieces + (STEP_U << spread) - 1) / (STEP_U << spread));
        const size_t grid = (((n * parts) << spread) + BLOCK - 1) / BLOCK;
        if (grid > 0x7fffffffull) return ERR_INVALID;
        gated_step_kernel<T, V, I><<<(unsigned)grid, BLOCK, 0, stream>>>(static_cast<const T*>(d_x), x_stride, static_cast<const T*>(d_gate), gate_stride, static_cast<float*>(d_state), pool,
                                                                       static_cast<const I*>(d_slots), n, pieces, spread, parts, static_cast<T*>(d_h));
        return (int)cudaGetLastError();
      };
      if (in_16_bytes(d_x, dim, x_stride, sizeof(T)) && in_16_bytes(d_gate, dim, gate_stride, sizeof(T)) && in_16_bytes(d_h, dim, dim, sizeof(T)) && in_16_bytes(d_state, dim, dim, 4))
        return go(std::integral_constant<int, 4>());
      return go(std::integral_constant<int, 1>());
    });
  });
}
