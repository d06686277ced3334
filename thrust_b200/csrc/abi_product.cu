// C ABI: tb200_expert_product, tb200_expert_product_grad and tb200_expert_activation_grad.
#include <cuda.h>
#include <type_traits>

#include "abi_rows.cuh"
#include "tensor_core.cuh"

using namespace tb200_abi;
using namespace tb200_rows;

namespace {
constexpr int MOST_EXPERTS = 1024;
constexpr size_t MOST_ROWS = (1ull << 31) - 1024, MOST_CHANNELS = 1ull << 24;

// ---------------------------------------------------------------------------------------------- activations
// silu(x) = x s(x) with s(x) = 1 / (1 + exp(-x)); gelu(x) = x P(x) with P the normal distribution.  s and 1 - s are made of exp(-|x|), which cannot overflow
// and keeps the smaller of the two good where it is tiny; P comes from erfc, which does not cancel where P is small.  FAST: s and P are good to a few 2^-22 (and
// 2^-24 |x|, 2^-23 x^2 for the exponential's argument) of themselves, for results that are rounded to 16 bits.
enum : int { ACT_NONE = TB200_ACT_NONE, ACT_SILU = TB200_ACT_SILU, ACT_GELU = TB200_ACT_GELU, ACT_GATED = TB200_ACT_GATED };
struct sigmoid_pair { float s, other; };
template <bool FAST> __device__ __forceinline__ sigmoid_pair sigmoid(float x) {
  float e, r;
  if (FAST) {
    asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * fabsf(x)));      // (not .ftz: exp(-88) is not zero)
    r = __fdividef(1.f, 1.f + e);
  } else {
    e = expf(-fabsf(x));
    r = 1.f / (1.f + e);
  }
  sigmoid_pair p;
  p.s = x >= 0.f ? r : e * r;
  p.other = x >= 0.f ? e * r : r;
  return p;
}
// P(x); FAST: from the Chebyshev fit of erfc in Numerical Recipes (Press et al., 6.2), good to 1.2e-7 of itself
template <bool FAST> __device__ __forceinline__ float normal_below(float x) {
  if (!FAST) return 0.5f * erfcf(-0.70710678118654752f * x);
  const float z = 0.70710678118654752f * fabsf(x), t = __fdividef(1.f, fmaf(0.5f, z, 1.f));
  float q = 0.17087277f;
  q = fmaf(q, t, -0.82215223f);
  q = fmaf(q, t, 1.48851587f);
  q = fmaf(q, t, -1.13520398f);
  q = fmaf(q, t, 0.27886807f);
  q = fmaf(q, t, -0.18628806f);
  q = fmaf(q, t, 0.09678418f);
  q = fmaf(q, t, 0.37409196f);
  q = fmaf(q, t, 1.00002368f);
  q = fmaf(q, t, -1.26551223f);
  float e;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(1.4426950408889634f * fmaf(-z, z, q)));
  const float tail = 0.5f * t * e;      // P(-|x|)
  return x >= 0.f ? 1.f - tail : tail;
}
template <bool FAST> __device__ __forceinline__ float activated(float x, int kind) { return kind == ACT_SILU ? x * sigmoid<FAST>(x).s : kind == ACT_GELU ? x * normal_below<FAST>(x) : x; }
// and with its slope
struct act_slope { float y, slope; };
template <bool FAST> __device__ __forceinline__ act_slope with_slope(float x, int kind) {
  if (kind == ACT_SILU) { const sigmoid_pair p = sigmoid<FAST>(x); return {x * p.s, p.s * fmaf(x, p.other, 1.f)}; }
  const float below = normal_below<FAST>(x);
  return {x * below, fmaf(x * 0.39894228040143268f, expf(-0.5f * x * x), below)};
}

// ---------------------------------------------------------------------------------------------- where the experts' rows are
// The offsets, cut off at the rows there are, and before each expert how many tiles of up to `tall` rows the experts before it have.
struct spans { int* at; int* tiles; };
__device__ __forceinline__ int read_offset(const void* offsets, bool wide, unsigned i, int m) {
  const long long o = wide ? static_cast<const long long*>(offsets)[i] : (long long)static_cast<const int*>(offsets)[i];
  return o < 0 ? 0 : o > m ? m : (int)o;
}
__device__ __forceinline__ int rows_of(const spans& s, unsigned e) { const int n = s.at[e + 1] - s.at[e]; return n > 0 ? n : 0; }
__device__ __forceinline__ void read_spans(spans s, const void* offsets, bool wide, unsigned experts, int m, int tall) {
  for (unsigned e = threadIdx.x; e <= experts; e += blockDim.x) s.at[e] = read_offset(offsets, wide, e, m);
  __syncthreads();
  if (threadIdx.x < 32) {
    int sum = 0;
    for (unsigned base = 0; base < experts; base += 32) {
      const unsigned e = base + threadIdx.x;
      const int own = e < experts ? (rows_of(s, e) + tall - 1) / tall : 0;
      const int upto = tb200::warp_inclusive_scan(own, tb200::plus_op());
      if (e < experts) s.tiles[e] = sum + upto - own;
      sum += __shfl_sync(tb200::FULL_MASK, upto, 31);
    }
    if (threadIdx.x == 0) s.tiles[experts] = sum;
  }
  __syncthreads();
}

// What one product is made of.  Features are what the lanes of a result's tile stand for, neighbours in memory; `others` what its columns stand for.
//   BY_ROWS: results are rows, a feature is an output, the contraction goes over k inputs.  BY_EXPERTS: a result is an expert's matrix, others x
//   features, and the contraction goes over the expert's rows.
enum : int { BY_ROWS, BY_EXPERTS };
template <class T> struct product_plan {
  const void* offsets;
  bool wide;
  unsigned experts;
  int m, k, features, others;
  int second;                 // gated: where the second half of the features begins in A
  bool a_mn;                  // A's features are neighbours (else its k)
  bool wide_out, wide_residual;      // rows are made of whole 16-byte pieces
  bool a_split, b_split;      // rows are made of whole chunks of 64 and mapped as such: a box has several
  int box;                    // by rows: rows in a box of B
  int planes;                 // 32-bit operands are three of 16 bits each, and six products of them are added up
  unsigned a_planes, b_planes;      // of which planes, two bits a segment
  const T *bias, *residual;
  size_t residual_stride;
  T *out, *before;
  int activation;
  void* matrix;
  bool accumulate, first;     // first: of the call's kernels, the one that clears the status; the others begin while those before them end
  tb200::ws_header* hdr;
};
struct product_tile { unsigned e; int row, rows, feature, other, depth; };

// Division by what is the same throughout a kernel: the upper half of a product with ceil(2^32 / d), which is the quotient or one more.
struct divisor {
  unsigned d, inverse;
  __device__ __forceinline__ explicit divisor(unsigned by) : d(by), inverse(by > 1 ? (unsigned)((0x100000000ull + by - 1) / by) : 0) {}
  __device__ __forceinline__ unsigned into(unsigned n, unsigned& rest) const {
    unsigned q = d > 1 ? __umulhi(n, inverse) : n;
    rest = n - q * d;
    if (rest >= d) { --q; rest += d; }      // (below zero)
    return q;
  }
};
// How tiles of WIDE features follow one another.
template <int MODE, int BN> struct tiling {
  divisor across, each;      // tiles of an index's features; by experts: tiles of an expert
  template <class T> __device__ __forceinline__ tiling(const product_plan<T>& p, int wide)
      : across((unsigned)(p.features + wide - 1) / wide), each(MODE == BY_ROWS ? 1u : across.d * ((unsigned)(p.others + BN - 1) / BN)) {}
};

// Tile t, asked for by whole warps.  By rows: an expert's rows in tiles of equal height (multiples of UNIT), all features of one before the next.  `e`: the expert of the
// last tile asked for, from which the search goes on, 32 experts at a time.
template <int MODE, int BN, int UNIT, class T>
__device__ __forceinline__ product_tile tile_at(const product_plan<T>& p, const spans& s, const tiling<MODE, BN>& g, int wide, unsigned t, unsigned& e) {
  product_tile r;
  unsigned in;
  if (MODE == BY_ROWS) {
    const unsigned index = g.across.into(t, in), lane = threadIdx.x % 32;
    for (unsigned found = 0; !found;) {
      const unsigned at = e + 1 + lane;
      found = __ballot_sync(tb200::FULL_MASK, index < (unsigned)s.tiles[at < p.experts ? at : p.experts]);
      e += found ? (unsigned)__ffs(found) - 1 : 32;
    }
    const int n = rows_of(s, e), parts = (n + BN - 1) / BN, tall = ((parts == 1 ? n : (n + parts - 1) / parts) + UNIT - 1) / UNIT * UNIT, part = (int)(index - s.tiles[e]);
    r.e = e;
    r.feature = (int)in * wide;
    r.row = s.at[e] + part * tall;
    r.rows = n - part * tall < tall ? n - part * tall : tall;
    r.other = 0;
    r.depth = p.k;
  } else {
    r.e = g.each.into(t, in);
    unsigned f;
    const unsigned o = g.across.into(in, f);
    r.feature = (int)f * wide;
    r.other = (int)o * BN;
    r.rows = p.others - r.other < BN ? p.others - r.other : BN;
    r.row = s.at[r.e];
    r.depth = rows_of(s, r.e);
  }
  return r;
}
template <int MODE, int WIDE, int BN, class T> __device__ __forceinline__ unsigned tiles_of(const product_plan<T>& p, const spans& s) {
  const unsigned across = (unsigned)(p.features + WIDE - 1) / WIDE;
  return MODE == BY_ROWS ? across * (unsigned)s.tiles[p.experts] : across * (unsigned)((p.others + BN - 1) / BN) * p.experts;
}
// Tiles are taken in turn by `takers`.  What is left over when all have had as many is cut into up to `most` parts each, as long as there are takers for them, so that the last
// turn is as much shorter: 536 tiles for 74 pairs take 7.3 turns instead of 8 (16382 f16 rows of 4096 to 2048 through eight experts: 243 us against 254).
struct turns {
  unsigned whole, parts, count;
  __device__ __forceinline__ turns(unsigned tiles, unsigned takers, unsigned most) {
    whole = tiles / takers * takers;
    const unsigned rest = tiles - whole;
    parts = rest ? takers / rest : 1;
    parts = parts > most ? most : parts;
    count = whole + rest * parts;
  }
  __device__ __forceinline__ unsigned tile(unsigned t) const { return t < whole || parts == 1 ? t : whole + (t - whole) / parts; }
  // of what a tile has of rows (by experts: of others); 0 where nothing is left for a part
  __device__ __forceinline__ void cut(unsigned t, int unit, int& first, int& rows) const {
    if (t < whole || parts == 1) return;
    const int part = (int)((t - whole) % parts), each = ((rows + (int)parts - 1) / (int)parts + unit - 1) / unit * unit;
    first += part * each;
    rows = rows - part * each < each ? rows - part * each : each;
    if (rows < 0) rows = 0;
  }
};

// rows [first, last) of `width` packed elements are zeros
template <class T> __device__ __forceinline__ void clear_rows(T* to, size_t first, size_t last, size_t width, size_t thread, size_t threads) {
  char* const begin = reinterpret_cast<char*>(to + first * width);
  char* const end = reinterpret_cast<char*>(to + last * width);
  char* const a = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(begin) + 15) & ~(uintptr_t)15);
  char* const b = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(end) & ~(uintptr_t)15);
  if (a >= b) {
    for (T* q = reinterpret_cast<T*>(begin) + thread; q < reinterpret_cast<T*>(end); q += threads) *q = from_f32<T>(0.f);
    return;
  }
  for (T* q = reinterpret_cast<T*>(begin) + thread; q < reinterpret_cast<T*>(a); q += threads) *q = from_f32<T>(0.f);
  for (T* q = reinterpret_cast<T*>(b) + thread; q < reinterpret_cast<T*>(end); q += threads) *q = from_f32<T>(0.f);
  for (uint4* q = reinterpret_cast<uint4*>(a) + thread; q < reinterpret_cast<uint4*>(b); q += threads) *q = make_uint4(0, 0, 0, 0);
}
// the rows that are no expert's
template <class T> __device__ __forceinline__ void clear_others(const product_plan<T>& p, const spans& s, size_t thread, size_t threads) {
  const size_t first = s.at[0], last = s.at[p.experts] > s.at[0] ? s.at[p.experts] : s.at[0], width = p.features, m = p.m;
  clear_rows(p.out, 0, first, width, thread, threads);
  clear_rows(p.out, last, m, width, thread, threads);
  if (p.before) {
    const size_t both = p.activation & ACT_GATED ? 2 * width : width;
    clear_rows(p.before, 0, first, both, thread, threads);
    clear_rows(p.before, last, m, both, thread, threads);
  }
}

// ---------------------------------------------------------------------------------------------- 16 bits: tensor cores
#ifdef TB200_TEST_HOOKS
// Test builds only: the copies of the first CTA's second tile are announced and not made, from stage withhold_boxes - 1 on.
__device__ unsigned withhold_boxes;
__device__ __forceinline__ bool withheld(unsigned t, unsigned step, int stage) { return withhold_boxes && blockIdx.x == 0 && t == step && (unsigned)stage + 1 >= withhold_boxes; }
#else
__device__ __forceinline__ bool withheld(unsigned, unsigned, int) { return false; }
#endif

constexpr int DEEP = 128;                     // of the contraction, a stage
// How many stages the matrix instructions add up; then the writers go on, with sums that are rounded to nearest.  See expert_product_kernel.
template <class O> constexpr int GROUP = sizeof(O) == 4 ? 6 : std::is_same<O, f16>::value ? 32 : 128;
// Warps: WRITERS that write results, then one that brings operands, one that multiplies, and (by experts) one that clears boxes' ends.  Few rows: four writers, and two CTAs a SM.
// 32-bit results: the writers hold 128 sums a thread, of registers that the other four warps hand over (launched with 168 a thread; 2 x 216 + 72 = 3 x 168).
template <int MODE, class O, bool PAIR> struct tc_warps {
  static constexpr bool FINE = sizeof(O) == 4, FEW = MODE == BY_ROWS && !PAIR && !FINE;
  static constexpr int WRITERS = FEW ? 4 : 8, THREADS = FINE ? 384 : (WRITERS + (MODE == BY_EXPERTS ? 3 : 2)) * 32, A_SM = FEW ? 2 : 1;
};
constexpr int WRITERS_REGISTERS = 216, OTHERS_REGISTERS = 72;
constexpr unsigned CHUNK = 64 * DEEP * 2;     // 64 neighbours by 128 of the other axis
constexpr unsigned A_BYTES = 2 * CHUNK;       // a CTA's 128 features

template <bool PAIR, int WRITERS, int BN, int STAGES> struct tc_shared {
  static constexpr unsigned B_CHUNK = BN * 128 / (PAIR ? 2 : 1), STAGE = A_BYTES + 2 * B_CHUNK, COLUMNS = 2 * BN;
  static_assert(COLUMNS <= 512, "two sets of sums in tensor memory");
  alignas(16) unsigned char turn[WRITERS][2048];      // where a writer's results are turned round
  unsigned long long full[STAGES], empty[STAGES], tail[STAGES], ready[STAGES], made[2], taken[2], done;
  unsigned tmem;
  int dead;
  static size_t bytes(unsigned experts) { return 1024 + (size_t)STAGES * STAGE + sizeof(tc_shared) + (2 * (size_t)experts + 2) * 4; }
};
// false: it did not come within the limit (of about a second), or another warp has given up.  stages: how many of the contraction it may have to wait for; 65536 of them
// take less than a tenth of the limit.
template <bool PAIR> __device__ __forceinline__ bool await(unsigned long long* bar, unsigned parity, int* dead, tb200::ws_header* hdr, unsigned stages = 0) {
  bool good = false;
  const unsigned long long limit = (unsigned long long)tb200::MBAR_SPIN_LIMIT * (1 + (stages >> 16));
  for (unsigned long long iter = 0; !good && iter < limit; ++iter) {
    good = PAIR ? tb200_tc::try_wait_pair(bar, parity) : tb200::mbar_try_wait(bar, parity);
    if (!good && *(volatile int*)dead) break;
  }
  good = __all_sync(tb200::FULL_MASK, good);
  if (!good && !*(volatile int*)dead) {
    *(volatile int*)dead = 1;
    tb200::record_error(&hdr->error, tb200::ERR_LOOKBACK_TIMEOUT);
  }
  return good;
}
// at the end, dead or not: what was asked for is not left on its way
__device__ __forceinline__ void outlast(unsigned long long* bar, unsigned parity) {
  for (unsigned iter = 0; iter < tb200::MBAR_SPIN_LIMIT && !tb200::mbar_try_wait(bar, parity); ++iter) {}
}

// Results of N columns in a lane's registers go to p, p + stride, ...; p: of the warp's first lane, whose neighbours' results lie next to its own.  With `wide` rows (whole
// 16-byte pieces) of a 16-bit type they are turned round in shared memory and written 16 bytes a lane, `room` elements (of 32) being there; otherwise element by element.
template <class O, int N> __device__ __forceinline__ void put_columns(O* p, size_t stride, int count, const float (&v)[N], int lane, int room, bool wide, unsigned char* turn) {
  if constexpr (sizeof(O) == 2) {
    if (wide) {
      O* const t = reinterpret_cast<O*>(turn);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < N; ++j) t[j * 32 + lane] = from_f32<O>(v[j]);
      __syncwarp();
      const int c = lane % 4 * 8;
#pragma unroll
      for (int i = 0; i < N / 8; ++i) {
        const int j = i * 8 + lane / 4;
        if (j < count && c < room) *reinterpret_cast<uint4*>(p + (size_t)j * stride + c) = *reinterpret_cast<const uint4*>(t + j * 32 + c);
      }
      return;
    }
  }
  if (lane >= room) return;
  p += lane;
  if (count >= N) {
#pragma unroll
    for (int j = 0; j < N; ++j) p[(size_t)j * stride] = from_f32<O>(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < count) p[(size_t)j * stride] = from_f32<O>(v[j]);
  }
}
// The same the other way: requested, and (turned round) added to v
template <class O, int N> struct columns_in {
  static constexpr int W = sizeof(O) == 2 ? N / 8 : 1;
  O at[N];
  uint4 pieces[W];
  __device__ __forceinline__ void request(const O* p, size_t stride, int count, int lane, int room, bool wide) {
    if constexpr (sizeof(O) == 2) {
      if (wide) {
        const int c = lane % 4 * 8;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const int j = i * 8 + lane / 4;
          if (j < count && c < room) pieces[i] = *reinterpret_cast<const uint4*>(p + (size_t)j * stride + c);
        }
        return;
      }
    }
    if (lane >= room || count <= 0) return;
    p += lane;
#pragma unroll
    for (int j = 0; j < N; ++j) at[j] = p[(size_t)(j < count ? j : count - 1) * stride];      // (no branch between the requests)
  }
  __device__ __forceinline__ void add(float (&v)[N], int lane, bool wide, unsigned char* turn) {
    if constexpr (sizeof(O) == 2) {
      if (wide) {
        O* const t = reinterpret_cast<O*>(turn);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(t)[i * 32 + lane] = pieces[i];
        __syncwarp();
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += to_f32(t[j * 32 + lane]);
        return;
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] += to_f32(at[j]);
  }
};

// A 32-bit number is a + b / 128 + c / 128^2 with three numbers of 16 bits (bf16), each the rest rounded: scaled by SCALE, rests of the smallest numbers are numbers of 16 bits too (2^-133
// is the least of them, so that c ends at 2^-147, where a 32-bit number's last bit is at 2^-149), and those of the largest, which would be rounded to infinity and are cut off instead, stay
// below it, with sums of products below the whole product.  Of the nine products of such planes the three smallest, 2^-24 of the whole together, are left out; the others are segments of
// one contraction, the smaller ones first: three of 1 / 128^2, two of 1 / 128, one of 1, and what is there is scaled as the next level begins.  (Six instructions for one, at fifteen times
// the rate of multiply-adds.)
constexpr int PLANES = 3, SEGMENTS = 6;
constexpr float SCALE = 128.f;
__host__ __device__ constexpr bool next_level(int segment) { return segment == 3 || segment == 5; }
constexpr unsigned A_PLANES = 2 | 0 << 2 | 1 << 4 | 1 << 6 | 0 << 8 | 0 << 10, B_PLANES = 0 | 2 << 2 | 1 << 4 | 0 << 6 | 1 << 8 | 0 << 10;

// D^T = A B^T by tiles of 128 features (gated: 64 of each half) a CTA x up to BN rows; CTAs stay and go from tile to tile.  Features are the lanes of tensor
// memory and rows its columns, so that a tile that has few rows takes a narrower instruction and no more time than they need: experts have as many rows as they have.
// PAIR: two CTAs have a tile of twice as many features, half of its rows' operands each, and instructions that read both's shared memory, which the first
// issues: 64 KB instead of 96 come from L2 for 256 features x 256 rows x 64.
//
// One warp keeps STAGES boxes of A and B on their way by the copy engine, one issues the matrix instructions as they come, the writers take the sums of the last
// tile from tensor memory, while the next one's are made in its other half, and write them.  Sums are 32 bits from first to last; they
// are rounded once, where they are stored, after bias, activation and residual.  The matrix instructions cut off what they add (of sums
// of one sign up to 1.5e-6 for each stage, and always the same way), so that they add up GROUP stages, and the writers add up those sums, rounded to nearest.  Results of 16 bits: 32 stages for
// f16 and 128 for bf16, which are off by 2.4e-5 and 9.6e-5, a tenth and a twentieth of the least half step; a longer contraction goes on in the other set, by way of the writers, which add
// the one to the other.  Sums of 2^20 numbers of one sign are off by half a step as those of 2^12 are (in one set: by 6e-3); 16384 f16 rows of 8192 to 512 take 142 us instead of 140,
// of 16384 234 instead of 225.  32-bit results (FINE) are made of sums over six stages, which the writers add up in registers,
// rounded to nearest, and put back to where the last ones were: off by 7.3e-7 in the norm (9.8e-7 where 2^20 are added up), twice that behind an activation that multiplies two
// results; with four stages 4.7e-7, and 8198 rows' gradients take 103 us instead of 98.  Gated: the two halves of a result are in lanes 64 apart, in warps that pass each
// other half of their columns.
//
// By experts the contraction ends where the expert's rows do, in the middle of a box: what the box has of the next rows is cleared in shared memory, up to
// the next 16, where the instructions end.  Such a box is counted by the barrier `tail` of the CTA that it is for, where a warp of its own clears it as soon as it is there and
// says that it is ready.
//
// Large products are bound by the power limit: 131072 bf16 rows of 2048 to 1536, gated, with what is kept, through 128 experts: 780 us (1020 TFLOP/s at 1.0 to 1.2 GHz, 79 % of the
// cycles the tensor cores'; without results written 680), 16382 f16 rows of 4096 to 2048 through eight 255 us (1080), 98304 rows' gradients 1024 to 2048 through 64
// 775 us for both products (1040).  Few rows are bound by the matrices' bytes: 132 rows of 2048 to 2048 through 64 experts 76 us with the call (6200 GB/s).  What had
// counted before: asking for boxes and issuing instructions lane by lane (950 us for the first), stages of 64 (884), single CTAs with tiles of 128 x 256 (951).
template <class T, class O, int MODE, bool PAIR, bool GATED, int BN, int STAGES>
__global__ void __launch_bounds__(tc_warps<MODE, O, PAIR>::THREADS, tc_warps<MODE, O, PAIR>::A_SM) expert_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const product_plan<T> p) {
  using Warps = tc_warps<MODE, O, PAIR>;
  constexpr int WRITERS = Warps::WRITERS, BRINGS = WRITERS, MULTIPLIES = WRITERS + 1, CLEARS = WRITERS + 2, APART = WRITERS * 8;
  using Shared = tc_shared<PAIR, WRITERS, BN, STAGES>;
  constexpr int CTAS = PAIR ? 2 : 1, OWN = GATED ? 64 : 128, WIDE = OWN * CTAS, UNIT = 16 * CTAS;
  constexpr bool FINE = Warps::FINE;
  constexpr int SEGS = sizeof(T) == 4 ? SEGMENTS : 1, LEVELS = sizeof(T) == 4 ? 3 : 1;      // (32-bit rows come here as planes)
  extern __shared__ char raw[];
  char* const stages = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  Shared& sh = *reinterpret_cast<Shared*>(stages + STAGES * Shared::STAGE);
  spans s;
  s.at = reinterpret_cast<int*>(&sh + 1);
  s.tiles = s.at + p.experts + 1;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  tb200::grid_dependents_launch();
  const unsigned rank = PAIR ? tb200_tc::rank_in_pair() : 0;
  if (threadIdx.x == 0) {
    if (blockIdx.x == 0 && p.first) p.hdr->error = 0;      // a wait that runs out does so long after this
    for (int i = 0; i < STAGES; ++i) {
      for (unsigned long long* bar : {&sh.full[i], &sh.empty[i], &sh.tail[i]}) tb200::mbar_init(bar, 1);
      tb200::mbar_init(&sh.ready[i], CTAS);
    }
    for (int i = 0; i < 2; ++i) { tb200::mbar_init(&sh.made[i], 1); tb200::mbar_init(&sh.taken[i], WRITERS * CTAS); }
    tb200::mbar_init(&sh.done, 1);
    sh.dead = 0;
    tb200::mbar_init_fence();
  }
  if (warp == MULTIPLIES) tb200_tc::tmem_alloc<PAIR>(&sh.tmem, Shared::COLUMNS);
  tb200_tc::fence_before_sync();
  read_spans(s, p.offsets, p.wide, p.experts, p.m, BN);
  if (PAIR) tb200_tc::meet_pair();
  tb200_tc::fence_after_sync();
  const unsigned tmem = sh.tmem, step = gridDim.x / CTAS;
  const turns turn(tiles_of<MODE, WIDE, BN>(p, s), step, MODE == BY_ROWS ? 4 : 2);
  const tiling<MODE, BN> follow(p, WIDE);
  // columns of a tile's instructions; of these each CTA brings its share of B
  const int unit = MODE == BY_EXPERTS && p.b_split ? 64 * CTAS : UNIT;
  auto columns_of = [&](const product_tile& tile) { return (tile.rows + unit - 1) / unit * unit; };
  auto tile_of = [&](unsigned t, unsigned& e) {
    product_tile tile = tile_at<MODE, BN, UNIT>(p, s, follow, WIDE, turn.tile(t), e);
    turn.cut(t, unit, MODE == BY_ROWS ? tile.row : tile.other, tile.rows);
    return tile;
  };
  auto is_tail = [&](const product_tile& tile, int k) { return MODE == BY_EXPERTS && tile.depth - k < DEEP && tile.depth % 16 != 0; };
  // what a box has beyond the expert's rows
  auto clear_tail = [&](unsigned stage, int valid, int boxes) {
    const int pieces = (16 - valid % 16) * 8;
    for (int i = lane; i < pieces * boxes; i += 32)
      *reinterpret_cast<uint4*>(stages + stage * Shared::STAGE + i / pieces * CHUNK + valid * 128 + i % pieces * 16) = make_uint4(0, 0, 0, 0);
    tb200::fence_async_smem();
    __syncwarp();
  };

  if (warp >= WRITERS) {
    static_assert(2 * WRITERS_REGISTERS + OTHERS_REGISTERS == 3 * 168, "no more registers than the CTA was launched with");
    if constexpr (FINE) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHERS_REGISTERS));
    if (warp == BRINGS) {
      const unsigned base = tb200::smem_addr(stages);
      unsigned count = 0, e = 0;      // stages filled so far
      bool good = true;
      for (unsigned t = blockIdx.x / CTAS; good && t < turn.count; t += step) {
        const product_tile tile = tile_of(t, e);
        if (tile.rows == 0) continue;
        const int share = columns_of(tile) / CTAS, feature = tile.feature + (int)rank * OWN, other = (MODE == BY_ROWS ? tile.row : tile.other) + (int)rank * share;
        // by rows B has two chunks of k, each of boxes of rows, unless a box has both; by experts two chunks of others, unless a box has both
        const int boxes = MODE == BY_ROWS ? (share + p.box - 1) / p.box : p.b_split ? 2 : (share + 63) / 64;
        const unsigned b_box = MODE == BY_ROWS ? p.box * 128 : CHUNK, bytes = A_BYTES + (MODE == BY_ROWS ? 2 : 1) * boxes * b_box;
        for (int k = 0, segment = 0; k < tile.depth; ++count) {
          const unsigned stage = count % STAGES, to = base + stage * Shared::STAGE;
          good = await<PAIR>(&sh.empty[stage], (count / STAGES & 1) ^ 1, &sh.dead, p.hdr);
          if (!good) break;
          const bool tail = is_tail(tile, k);
          if (tb200_tc::elected()) {
            unsigned bar;
            if (tail) {
              tb200::mbar_arrive_expect(&sh.tail[stage], bytes);
              if (rank == 0) tb200::mbar_arrive(&sh.full[stage]);
              bar = tb200::smem_addr(&sh.tail[stage]);
            } else {
              if (rank == 0) tb200::mbar_arrive_expect(&sh.full[stage], bytes * CTAS);
              bar = PAIR ? tb200_tc::first_ones(&sh.full[stage]) : tb200::smem_addr(&sh.full[stage]);
            }
            if (!withheld(t, step, k / DEEP)) {
              const int row = MODE == BY_ROWS ? k : tile.row + k, pa = (int)(p.a_planes >> 2 * segment & 3), pb = (int)(p.b_planes >> 2 * segment & 3);
              const int of_a = MODE == BY_ROWS ? (int)tile.e * p.planes + pa : pa;
              const bool both = p.a_split || (GATED && p.a_mn);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                if (c && both) continue;
                tb200_tc::box_at at;
                if (MODE == BY_EXPERTS || p.a_mn) at = {p.a_split ? 0 : feature + c * 64, row, p.a_split ? feature / 64 : 0, 0, of_a};
                else at = {p.a_split ? 0 : k + c * 64, feature, p.a_split && !GATED ? k / 64 : 0, p.a_split && GATED ? k / 64 : 0, of_a};
                tb200_tc::load_box<PAIR>(to + c * CHUNK, &map_a, at, bar);
              }
              if (MODE == BY_EXPERTS) {
                if (p.b_split) tb200_tc::load_box<PAIR>(to + A_BYTES, &map_b, {0, row, other / 64, 0, pb}, bar);
                else
                  for (int b = 0; b < boxes; ++b) tb200_tc::load_box<PAIR>(to + A_BYTES + b * CHUNK, &map_b, {other + b * 64, row, 0, 0, pb}, bar);
              } else if (PAIR && p.b_split) {
                tb200_tc::load_box<PAIR>(to + A_BYTES, &map_b, {0, other, k / 64, 0, pb}, bar);
              } else {
                for (int c = 0; c < 2; ++c)
                  for (int b = 0; b < boxes; ++b) tb200_tc::load_box<PAIR>(to + A_BYTES + c * Shared::B_CHUNK + b * b_box, &map_b, {k + c * 64, other + b * p.box, 0, 0, pb}, bar);
              }
            }
          }
          __syncwarp();
          if ((k += DEEP) >= tile.depth && ++segment < SEGS) k = 0;
        }
      }
      // the last of each stage, no longer needed
      if (good)
        for (unsigned i = 0; i < STAGES && i < count; ++i) good = good && await<PAIR>(&sh.empty[(count - 1 - i) % STAGES], (count - 1 - i) / STAGES & 1, &sh.dead, p.hdr);
      // given up: what is on its way is counted where this warp may not be able to see it; copies take microseconds
      if (!good)
        for (int i = 0; i < 20; ++i) __nanosleep(1000000);
    } else if (warp == MULTIPLIES) {
      const unsigned base = tb200::smem_addr(stages);
      unsigned count = 0, made = 0, e = 0, tails = 0;      // tails: a bit for each stage's barrier
      bool good = true;
      const bool a_mn = MODE == BY_EXPERTS || p.a_mn;
      constexpr bool b_mn = MODE == BY_EXPERTS;
      // from one 16 k to the next, and from one 64 to the next, in a descriptor's units of 16 bytes
      const unsigned a_step = a_mn ? 16 * 128 >> 4 : 2, a_jump = a_mn ? 64 * 128 >> 4 : CHUNK >> 4;
      constexpr unsigned b_step = b_mn ? 16 * 128 >> 4 : 2, b_jump = b_mn ? 64 * 128 >> 4 : Shared::B_CHUNK >> 4;
      if (rank == 0) {
        for (unsigned t = blockIdx.x / CTAS; good && t < turn.count; t += step) {
          const product_tile tile = tile_of(t, e);
          if (tile.depth == 0 || tile.rows == 0) continue;
          const unsigned what = tb200_tc::instruction<PAIR>(!std::is_same<T, f16>::value, a_mn, b_mn, columns_of(tile));
          unsigned set = 0, d = 0;
          bool begun = false;      // these sums are
          for (int k = 0, segment = 0, block = 0; k < tile.depth; ++count) {
            if (!begun) {
              set = made & 1;
              d = tmem + set * BN;
              good = await<PAIR>(&sh.taken[set], (made / 2 & 1) ^ 1, &sh.dead, p.hdr);
              if (!good) break;
              ++made;
              tb200_tc::fence_after_sync();
            }
            const unsigned stage = count % STAGES, from = base + stage * Shared::STAGE;
            good = await<PAIR>(&sh.full[stage], count / STAGES & 1, &sh.dead, p.hdr);
            if (!good) break;
            const int valid = tile.depth - k < DEEP ? tile.depth - k : DEEP, steps = (valid + 15) / 16;
            if (is_tail(tile, k)) {
              good = await<PAIR>(&sh.ready[stage], tails >> stage & 1, &sh.dead, p.hdr);
              if (!good) break;
              tails ^= 1u << stage;
            }
            tb200_tc::fence_after_sync();
            if (tb200_tc::elected()) {
              const unsigned long long a = tb200_tc::operand(from, a_mn, CHUNK), b = tb200_tc::operand(from + A_BYTES, b_mn, CHUNK);
#pragma unroll
              for (int i = 0; i < DEEP / 16; ++i)
                if (i < steps) tb200_tc::multiply<PAIR>(d, a + i / 4 * a_jump + i % 4 * a_step, b + i / 4 * b_jump + i % 4 * b_step, what, begun || i > 0);
              tb200_tc::commit<PAIR>(&sh.empty[stage]);
            }
            __syncwarp();
            begun = true;
            bool cut = ++block == GROUP<O>;
            if ((k += DEEP) >= tile.depth) {
              if (++segment < SEGS) k = 0;
              cut = cut || segment == SEGS || next_level(segment);
            }
            if (cut) {
              block = 0;
              if (tb200_tc::elected()) tb200_tc::commit<PAIR>(&sh.made[set]);
              __syncwarp();
              begun = false;
            }
          }
        }
        if (tb200_tc::elected()) { tb200_tc::commit_here<PAIR>(&sh.done); outlast(&sh.done, 0); }
        __syncwarp();
      }
    } else if (MODE == BY_EXPERTS && warp == CLEARS) {
      unsigned count = 0, e = 0, tails = 0;
      bool good = true;
      for (unsigned t = blockIdx.x / CTAS; good && t < turn.count; t += step) {
        const product_tile tile = tile_of(t, e);
        if (tile.rows == 0) continue;
        const unsigned blocks = (unsigned)(tile.depth + DEEP - 1) / DEEP;
        const bool has = blocks > 0 && is_tail(tile, (int)(blocks - 1) * DEEP);
        for (int segment = 0; good && segment < SEGS; ++segment) {
          const unsigned stage = (count + blocks - 1) % STAGES;
          count += blocks;
          if (!has) continue;
          good = await<PAIR>(&sh.tail[stage], tails >> stage & 1, &sh.dead, p.hdr, 2 * blocks);
          if (!good) break;
          tails ^= 1u << stage;
          clear_tail(stage, tile.depth - (int)(blocks - 1) * DEEP, 2 + (columns_of(tile) / CTAS + 63) / 64);
          if (lane == 0) {
            if (PAIR) tb200_tc::arrive_there(tb200_tc::first_ones(&sh.ready[stage]));
            else tb200::mbar_arrive(&sh.ready[stage]);
          }
          __syncwarp();
        }
      }
    }
  } else {
    if constexpr (FINE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(WRITERS_REGISTERS));
    // a writer has the 32 lanes that warp % 4 may read, and 32 columns of every APART; GATED: of these it finishes 16, of both halves
    unsigned made = 0, e = 0;
    bool good = true;
    const int kind = p.activation & ~ACT_GATED, quarter = warp % 4, half = GATED ? quarter / 2 : 0, within = (GATED ? quarter % 2 : quarter) * 32;
    unsigned char* const room_of = sh.turn[warp];
    constexpr int PUT = GATED ? 16 : 32;
    for (unsigned t = blockIdx.x / CTAS; t < turn.count; t += step) {
      const product_tile tile = tile_of(t, e);
      if (tile.rows == 0) continue;
      const int f = tile.feature + (int)rank * OWN + within, room = p.features - f;      // the first lane's feature, and how many there are from there on
      const bool there = lane < room;
      const size_t width = p.features, both = GATED ? 2 * width : width;
      float bias = 0.f;
      if (MODE == BY_ROWS && p.bias && there) bias = to_f32(p.bias[tile.e * both + half * width + f + lane]);
      columns_in<T, PUT> residual;
      columns_in<O, 32> old;
      // what results of columns c on are added to is asked for
      auto request = [&](int c) {
        const int mine = c + half * 16;
        if (c >= tile.rows) return;
        if (MODE == BY_ROWS && p.residual)
          residual.request(p.residual + ((size_t)tile.row + mine) * p.residual_stride + f, p.residual_stride, tile.rows - mine, lane, room, p.wide_residual);
        if (MODE == BY_EXPERTS && p.accumulate && tile.depth)
          old.request(static_cast<O*>(p.matrix) + ((size_t)tile.e * p.others + tile.other + c) * width + f, width, tile.rows - c, lane, room, p.wide_out);
      };
      // the sums of 32 columns become results
      auto finish = [&](int c, float (&v)[32]) {
        const int mine = c + half * 16;
        if constexpr (MODE == BY_ROWS) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += bias;
          if (p.before) put_columns(p.before + ((size_t)tile.row + c) * both + half * width + f, both, tile.rows - c, v, lane, room, p.wide_out, room_of);
          float w[PUT];
          if constexpr (GATED) {
            float (&out)[16][32] = *reinterpret_cast<float(*)[16][32]>(room_of), (&in)[16][32] = *reinterpret_cast<float(*)[16][32]>(sh.turn[warp ^ 2]);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j) out[j][lane] = half ? v[j] : v[j + 16];
            const int pair = 1 + warp / 4 * 2 + warp % 2;      // the barrier of the two warps
            asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
#pragma unroll
            for (int j = 0; j < 16; ++j) { const float x = in[j][lane]; w[j] = half ? x : v[j]; v[j] = half ? v[j + 16] : x; }      // act(w) v
            asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory");
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) w[j] = v[j];
          }
#pragma unroll
          for (int part = 0; part < PUT; part += 8) {      // (few rows: not for columns that are not there)
            if (mine + part >= tile.rows) break;
            if (kind == ACT_SILU) {
#pragma unroll
              for (int j = part; j < part + 8; ++j) w[j] = activated<sizeof(T) == 2>(w[j], ACT_SILU);
            } else if (kind == ACT_GELU) {
#pragma unroll
              for (int j = part; j < part + 8; ++j) w[j] = activated<sizeof(T) == 2>(w[j], ACT_GELU);
            }
          }
          if constexpr (GATED) {
#pragma unroll
            for (int j = 0; j < PUT; ++j) w[j] *= v[j];
          }
          if (p.residual) residual.add(w, lane, p.wide_residual, room_of);
          put_columns(p.out + ((size_t)tile.row + mine) * width + f, width, tile.rows - mine, w, lane, room, p.wide_out, room_of);
        } else {
          O* const to = static_cast<O*>(p.matrix) + ((size_t)tile.e * p.others + tile.other + c) * width + f;
          if (p.accumulate && tile.depth == 0 && good) return;      // (an expert without rows adds nothing)
          if (p.accumulate) old.add(v, lane, p.wide_out, room_of);
          put_columns(to, width, tile.rows - c, v, lane, room, p.wide_out, room_of);
        }
      };
      auto await_sums = [&] {
        if (good) good = await<PAIR>(&sh.made[made & 1], made / 2 & 1, &sh.dead, p.hdr);
        tb200_tc::fence_after_sync();
      };
      auto set_free = [&](unsigned set) {      // the next sums may be made there
        tb200_tc::fence_before_sync();
        __syncwarp();
        if (lane == 0 && good) {
          if (PAIR) tb200_tc::arrive_there(tb200_tc::first_ones(&sh.taken[set]));
          else tb200::mbar_arrive(&sh.taken[set]);
        }
      };
      auto sums_taken = [&] { set_free(made++ & 1); };
      const unsigned lanes = quarter * 32u << 16;
      bool waited = tile.depth == 0;
      const int blocks = (tile.depth + DEEP - 1) / DEEP;
      auto groups_of = [&](int segments) { return (blocks * segments + GROUP<O> - 1) / GROUP<O>; };
      if constexpr (!FINE) {
        // each group's sums are added to those of all before it, in the other set, which the group after it may then have
        for (int g = 0; g + 1 < groups_of(1); ++g) {
          if (g == 0) await_sums();
          ++made;
          await_sums();
          const unsigned at = tmem + lanes + (made & 1) * BN, before = tmem + lanes + (~made & 1) * BN;
          for (int c = warp / 4 * 32; c < tile.rows && good; c += APART) {
            float v[32], sums[32];
            tb200_tc::tmem_load(sums, before + c);
            tb200_tc::tmem_load(v, at + c);
            tb200_tc::tmem_load_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += sums[j];
            tb200_tc::tmem_store(v, at + c);
          }
          tb200_tc::tmem_store_wait();
          set_free(~made & 1);
          waited = true;
        }
      } else {
        // the sums of all groups, added up in registers, take the last one's place
        constexpr int N = BN / APART;
        if (tile.depth && (LEVELS > 1 || groups_of(1) > 1)) {
          float sums[N][32];
#pragma unroll
          for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 32; ++j) sums[i][j] = 0.f;
          for (int level = LEVELS; level > 0; --level) {      // so many segments have its scale
            const int groups = groups_of(level);
            for (int g = 0; g < groups; ++g) {
              const float scale = g == 0 && level < LEVELS ? 1.f / SCALE : 1.f;
              await_sums();
#pragma unroll
              for (int i = 0; i < N; ++i) {
                const int c = warp / 4 * 32 + i * APART;
                if (c >= tile.rows || !good) continue;
                float v[32];
                tb200_tc::tmem_load(v, tmem + lanes + (made & 1) * BN + c);
                tb200_tc::tmem_load_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) sums[i][j] = fmaf(sums[i][j], scale, v[j]);
              }
              if (level > 1 || g + 1 < groups) sums_taken();
            }
          }
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (warp / 4 * 32 + i * APART < tile.rows) tb200_tc::tmem_store(sums[i], tmem + lanes + (made & 1) * BN + warp / 4 * 32 + i * APART);
          tb200_tc::tmem_store_wait();
          waited = true;
        }
      }
      for (int c = warp / 4 * 32;; c += APART) {
        const bool any = c < tile.rows, last = c + APART >= tile.rows;
        request(c);
        if (!waited) await_sums();
        waited = true;
        float v[32];
        if (any && tile.depth && good) {
          tb200_tc::tmem_load(v, tmem + lanes + (made & 1) * BN + c);
          tb200_tc::tmem_load_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = good ? 0.f : __int_as_float(0x7fffffff);
        }
        if (last && tile.depth) sums_taken();
        if (any) finish(c, v);
        if (last) break;
      }
    }
    if (MODE == BY_ROWS) clear_others(p, s, (size_t)blockIdx.x * WRITERS * 32 + threadIdx.x, (size_t)gridDim.x * WRITERS * 32);
    tb200_tc::fence_before_sync();
  }
  __syncthreads();
  tb200::grid_dependency_wait();      // (nothing here needs what ran before, but what comes after may)
  if (PAIR) tb200_tc::meet_pair();      // neither ends while the other's instructions and arrivals come here
  if (warp == MULTIPLIES) {
    tb200_tc::fence_after_sync();
    tb200_tc::tmem_free<PAIR>(tmem, Shared::COLUMNS);
  }
}

// ---------------------------------------------------------------------------------------------- 32 bits: fused multiply-adds
// Products of 32-bit rows are made by the ordinary units: the matrix instructions round their operands to 11 bits or fewer.  Tiles of 128 features (gated: 64
// of each half) x BN rows; a lane has 2 FP features x 8 rows, eight lanes by four, two features side by side in its multiply-adds (f32x2).  Operands go 16 bytes at a time,
// by asynchronous copies, into a ring of stages of shared memory, and lie there as they lie in memory: by k (rows of features or of others), or by m (rows of
// k), of which a lane takes two k at a time.  Bound by the multiply-adds: 2048 rows of 1000 to 1501 through six experts took 176 us (35 TFLOP/s; tiles of
// 128 x 128 read element by element 298), which the tensor cores take 61 for.  They have the products of few rows and of few channels.
//
// One multiply-add after another rounds a sum each time: FMA_GROUP stages (1024 of the contraction) are added up that way, and those sums to one another, so that 500000 rows of one
// expert's gradient are off by 3e-7 in the norm (one after another: 9e-6), whatever the other experts have.
constexpr int FMA_THREADS = 128, FMA_DEEP = 16, FMA_STAGES = 4, FMA_GROUP = 64;
template <int WIDE, bool BY_K> struct fma_tile {      // an operand's part of a stage
  static constexpr int STRIDE = BY_K ? WIDE + 4 : FMA_DEEP + 4, PIECES = WIDE * FMA_DEEP / 4 / FMA_THREADS;
  float at[(BY_K ? FMA_DEEP : WIDE) * STRIDE];
};
template <int MODE, bool A_MN, int BN> struct fma_shared {
  static constexpr bool A_BY_K = MODE == BY_EXPERTS || A_MN, B_BY_K = MODE == BY_EXPERTS;
  fma_tile<128, A_BY_K> a[FMA_STAGES];
  fma_tile<BN, B_BY_K> b[FMA_STAGES];
  static size_t bytes(unsigned experts) { return sizeof(fma_shared) + (2 * (size_t)experts + 2) * 4; }
};
// 16 bytes on their way to shared memory, of which `words` are there; zero for the others
__device__ __forceinline__ void copy_words(float* to, const float* from, int words) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tb200::smem_addr(to)), "l"(from), "r"(words * 4) : "memory");
}
__device__ __forceinline__ int within_four(int n) { return n < 0 ? 0 : n > 4 ? 4 : n; }
using f2 = unsigned long long;
__device__ __forceinline__ f2 pack2(float x, float y) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y)); return r; }
__device__ __forceinline__ float2 unpack2(f2 a) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a)); return r; }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }

template <int MODE, bool A_MN, int BN>
__global__ void __launch_bounds__(FMA_THREADS, 3) expert_product_f32_kernel(const float* __restrict__ a, size_t a_expert, size_t a_stride, const float* __restrict__ b, size_t b_stride,
                                                                            const product_plan<float> p) {
  using Shared = fma_shared<MODE, A_MN, BN>;
  constexpr bool A_BY_K = Shared::A_BY_K, B_BY_K = Shared::B_BY_K;
  constexpr int FP = BN == 64 ? 4 : 2, ACROSS = 64 / (8 * FP), SA = fma_tile<128, A_BY_K>::STRIDE, SB = fma_tile<BN, B_BY_K>::STRIDE;
  extern __shared__ __align__(16) char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  spans s;
  s.at = reinterpret_cast<int*>(&sh + 1);
  s.tiles = s.at + p.experts + 1;
  if (threadIdx.x == 0 && blockIdx.x == 0 && p.first) p.hdr->error = 0;      // nothing here waits
  read_spans(s, p.offsets, p.wide, p.experts, p.m, BN);
  const bool gated = MODE == BY_ROWS && (p.activation & ACT_GATED);
  // tiles are as wide as the features they have: half as wide where they are of two halves
  const unsigned across = (unsigned)(p.features + (gated ? 63 : 127)) / (gated ? 64 : 128);
  const unsigned tiles = gated ? across * (unsigned)s.tiles[p.experts] : tiles_of<MODE, 128, BN>(p, s);
  const tiling<MODE, BN> follow(p, gated ? 64 : 128);
  // this lane's features (of either 64) and rows
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, x0 = warp % ACROSS * 8 * FP, y0 = warp / ACROSS * 32;
  auto x_of = [&](int i) { return x0 + (A_BY_K ? lane % 8 * FP + i : lane % 8 + 8 * i); };
  auto y_of = [&](int j) { return y0 + (B_BY_K ? lane / 8 * 4 + j % 4 + j / 4 * 16 : lane / 8 + 4 * j); };
  unsigned e = 0;
  for (unsigned t = blockIdx.x; t < tiles; t += gridDim.x) {
    const product_tile tile = tile_at<MODE, BN, 1>(p, s, follow, gated ? 64 : 128, t, e);
    if (MODE == BY_EXPERTS && tile.depth == 0 && p.accumulate) continue;      // nothing is added
    const int wide = p.features - tile.feature < (gated ? 64 : 128) ? p.features - tile.feature : gated ? 64 : 128;      // features of the tile, gated of either half
    // this thread's pieces of a stage: where they lie in the tile, where the first comes from (at k = 0), of A also the first of the upper 64 features
    constexpr int PA = fma_tile<128, A_BY_K>::PIECES, PB = fma_tile<BN, B_BY_K>::PIECES;
    const int ka = A_BY_K ? threadIdx.x / 32 : threadIdx.x % 4 * 4, wa = A_BY_K ? threadIdx.x % 32 * 4 : threadIdx.x / 4;
    const int kb = B_BY_K ? threadIdx.x / (BN / 4) : threadIdx.x % 4 * 4, wb = B_BY_K ? threadIdx.x % (BN / 4) * 4 : threadIdx.x / 4;
    constexpr int A_K = A_BY_K ? 4 : 0, A_W = A_BY_K ? 0 : 32, B_K = B_BY_K ? FMA_THREADS * 4 / BN : 0, B_W = B_BY_K ? 0 : 32;      // from one piece to the next
    auto column_of = [&](int w) { return (size_t)tile.feature + (gated && w >= 64 ? p.second + w - 64 : w); };
    auto left_of = [&](int w) { return wide - (gated && w >= 64 ? w - 64 : w); };      // features from w on
    const float *a0, *a1;
    if (A_BY_K) {
      a0 = a + (MODE == BY_ROWS ? tile.e * a_expert : (size_t)tile.row * a_stride) + (size_t)ka * a_stride + column_of(wa);
      a1 = a0;
    } else {
      a0 = a + tile.e * a_expert + column_of(wa) * a_stride + ka;
      a1 = a + tile.e * a_expert + column_of(wa + 64) * a_stride + ka;
    }
    const float* b0 = B_BY_K ? b + ((size_t)tile.row + kb) * b_stride + tile.other + wb : b + ((size_t)tile.row + wb) * b_stride + kb;
    auto fetch = [&](int k0, int stage) {
#pragma unroll
      for (int i = 0; i < PA; ++i) {
        const int k = ka + i * A_K, w = wa + i * A_W;
        const int words = A_BY_K ? (k0 + k < tile.depth ? within_four(left_of(w)) : 0) : left_of(w) > 0 ? within_four(tile.depth - k0 - k) : 0;
        const float* const from = A_BY_K ? a0 + (size_t)(i * A_K) * a_stride : (i < 2 ? a0 : a1) + (size_t)(i % 2 * A_W) * a_stride;
        copy_words(&sh.a[stage].at[(A_BY_K ? k : w) * SA + (A_BY_K ? w : k)], words ? from : a, words);
      }
#pragma unroll
      for (int i = 0; i < PB; ++i) {
        const int k = kb + i * B_K, w = wb + i * B_W;
        const int words = B_BY_K ? (k0 + k < tile.depth ? within_four(tile.rows - w) : 0) : w < tile.rows ? within_four(tile.depth - k0 - k) : 0;
        const float* const from = b0 + (size_t)(B_BY_K ? i * B_K : i * B_W) * b_stride;
        copy_words(&sh.b[stage].at[(B_BY_K ? k : w) * SB + (B_BY_K ? w : k)], words ? from : b, words);
      }
      a0 += A_BY_K ? FMA_DEEP * a_stride : FMA_DEEP;
      a1 += A_BY_K ? FMA_DEEP * a_stride : FMA_DEEP;
      b0 += B_BY_K ? FMA_DEEP * b_stride : FMA_DEEP;
    };
    f2 acc[FP][8];      // pairs of the lower features, then of the upper
#pragma unroll
    for (int i = 0; i < FP; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i][j] = pack2(0.f, 0.f);
    volatile f2 all[FP * 8];      // sums of long contractions, in local memory
    const int blocks = (tile.depth + FMA_DEEP - 1) / FMA_DEEP;
    __syncthreads();      // (the last tile's stages have been read)
    for (int q = 0; q < FMA_STAGES - 1; ++q) {
      if (q < blocks) fetch(q * FMA_DEEP, q);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    for (int q = 0; q < blocks; ++q) {
      asm volatile("cp.async.wait_group %0;" ::"n"(FMA_STAGES - 2) : "memory");
      __syncthreads();
      if (q + FMA_STAGES - 1 < blocks) fetch((q + FMA_STAGES - 1) * FMA_DEEP, (q + FMA_STAGES - 1) % FMA_STAGES);
      asm volatile("cp.async.commit_group;" ::: "memory");
      const float *const sa = sh.a[q % FMA_STAGES].at, *const sb = sh.b[q % FMA_STAGES].at;
#pragma unroll
      for (int k = 0; k < FMA_DEEP; k += 2) {
        float2 xs[A_BY_K ? 1 : 2 * FP], ys[B_BY_K ? 1 : 8];      // two k of a feature, of a row
        if constexpr (!A_BY_K) {
#pragma unroll
          for (int i = 0; i < 2 * FP; ++i) xs[i] = *reinterpret_cast<const float2*>(sa + ((i < FP ? 0 : 64) + x_of(i % FP)) * SA + k);
        }
        if constexpr (!B_BY_K) {
#pragma unroll
          for (int j = 0; j < 8; ++j) ys[j] = *reinterpret_cast<const float2*>(sb + y_of(j) * SB + k);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f2 x[FP];
          float y[8];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float* const from = sa + (k + u) * SA + h * 64 + x_of(0);
            if constexpr (!A_BY_K) {
#pragma unroll
              for (int i = 0; i < FP / 2; ++i) {
                const float2 m = xs[h * FP + 2 * i], n = xs[h * FP + 2 * i + 1];
                x[h * FP / 2 + i] = u ? pack2(m.y, n.y) : pack2(m.x, n.x);
              }
            } else if constexpr (FP == 4) {
              *reinterpret_cast<ulonglong2*>(x + h * 2) = *reinterpret_cast<const ulonglong2*>(from);
            } else {
              x[h] = *reinterpret_cast<const f2*>(from);
            }
            if constexpr (B_BY_K) *reinterpret_cast<float4*>(y + h * 4) = *reinterpret_cast<const float4*>(sb + (k + u) * SB + y_of(h * 4));
          }
          if constexpr (!B_BY_K) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = u ? ys[j].y : ys[j].x;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const f2 both = pack2(y[j], y[j]);
#pragma unroll
            for (int f = 0; f < FP; ++f) acc[f][j] = fma2(x[f], both, acc[f][j]);
          }
        }
      }
      if (q % FMA_GROUP == FMA_GROUP - 1 && q + 1 < blocks) {
#pragma unroll
        for (int i = 0; i < FP; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            all[i * 8 + j] = q < FMA_GROUP ? acc[i][j] : add2(all[i * 8 + j], acc[i][j]);
            acc[i][j] = pack2(0.f, 0.f);
          }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (blocks > FMA_GROUP) {
#pragma unroll
      for (int i = 0; i < FP; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = add2(all[i * 8 + j], acc[i][j]);
    }
    const size_t width = p.features;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int n = y_of(j);
      if (n >= tile.rows) continue;
      const size_t row = (size_t)tile.row + n;
      float sums[2 * FP];
#pragma unroll
      for (int i = 0; i < FP; ++i) { const float2 v = unpack2(acc[i][j]); sums[2 * i] = v.x; sums[2 * i + 1] = v.y; }
#pragma unroll
      for (int i = 0; i < 2 * FP; ++i) {
        if (gated && i >= FP) continue;
        const int f = tile.feature + (i < FP ? 0 : 64) + x_of(i % FP);
        if (f >= p.features) continue;
        float v = sums[i];
        if (MODE == BY_ROWS) {
          const int kind = p.activation & ~ACT_GATED;
          const size_t both = gated ? 2 * width : width;
          float u = sums[i < FP ? i + FP : i];
          if (p.bias) { v += p.bias[tile.e * both + f]; if (gated) u += p.bias[tile.e * both + width + f]; }
          if (p.before) { p.before[row * both + f] = v; if (gated) p.before[row * both + width + f] = u; }
          v = activated<false>(v, kind);
          if (gated) v *= u;
          if (p.residual) v += p.residual[row * p.residual_stride + f];
          p.out[row * width + f] = v;
        } else {
          float* const q = static_cast<float*>(p.matrix) + ((size_t)tile.e * p.others + tile.other + n) * width + f;
          *q = p.accumulate ? *q + v : v;
        }
      }
    }
  }
  if (MODE == BY_ROWS) clear_others(p, s, (size_t)blockIdx.x * FMA_THREADS + threadIdx.x, (size_t)gridDim.x * FMA_THREADS);
}

// ---------------------------------------------------------------------------------------------- the smaller parts
// The gradient of bias: the sums of each expert's rows of dout.  A CTA has 32 V features of one of `parts` pieces of an expert's rows; its warps take rows in turn and
// meet in shared memory, parts meet in a second kernel, always in the same order.  Bound by latency: 8198 bf16 rows of 1280 for 16 experts 10 us and 4, beside the products.
// SUM_GROUP rows, of which a warp adds up 1024, make a sum of their own: how many parts there are goes by the rows of an expert on average, and one expert may have nearly all
// (4000000 rows of numbers of one sign: off by 7.7e-8, in chains of 250000 by 1.5e-6).
constexpr int SUM_BLOCK = 256, SUM_GROUP = 1024 * SUM_BLOCK / 32;
template <class T, int V>
__global__ void __launch_bounds__(SUM_BLOCK) row_sums_kernel(const T* __restrict__ x, size_t stride, const void* __restrict__ offsets, bool wide, unsigned experts, int m, int features,
                                                             float* __restrict__ sums, tb200::ws_header* hdr) {
  const unsigned e = blockIdx.y, part = blockIdx.z, parts = gridDim.z;
  const int a = read_offset(offsets, wide, e, m), end = read_offset(offsets, wide, e + 1, m), n = end > a ? end - a : 0, per = (n + (int)parts - 1) / (int)parts;
  const int first = a + (int)part * per, last = (int)part * per + per < n ? first + per : a + n;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, f = (blockIdx.x * 32 + lane) * V;
  tb200::grid_dependents_launch();
  if (hdr && threadIdx.x == 0 && blockIdx.x + blockIdx.y + blockIdx.z == 0) hdr->error = 0;      // no product has cleared it, and nothing here waits
  float sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) sum[v] = 0.f;
  for (int begin = first; f < features && begin < last;) {
    const int stop = last - begin > SUM_GROUP ? begin + SUM_GROUP : last;
    float some[V];
#pragma unroll
    for (int v = 0; v < V; ++v) some[v] = 0.f;
#pragma unroll 4
    for (int r = begin + warp; r < stop; r += SUM_BLOCK / 32) {
      float g[V];
      channels(load_words<T, V>(x + (size_t)r * stride + f), g);
#pragma unroll
      for (int v = 0; v < V; ++v) some[v] += g[v];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] += some[v];
    begin = stop;
  }
  __shared__ float met[SUM_BLOCK / 32][32 * V];
#pragma unroll
  for (int v = 0; v < V; ++v) met[warp][lane * V + v] = sum[v];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += SUM_BLOCK) {
    const int g = blockIdx.x * 32 * V + i;
    if (g >= features) break;
    float all = 0.f;
#pragma unroll
    for (int w = 0; w < SUM_BLOCK / 32; ++w) all += met[w][i];
    sums[((size_t)part * experts + e) * features + g] = all;
  }
  tb200::grid_dependency_wait();      // (as the products': what comes after waits for them too)
}
__global__ void __launch_bounds__(SUM_BLOCK) join_sums_kernel(const float* __restrict__ sums, size_t items, unsigned parts, float* __restrict__ out) {
  const size_t i = (size_t)blockIdx.x * SUM_BLOCK + threadIdx.x;
  tb200::grid_dependency_wait();
  if (i >= items) return;
  float sum = 0.f;
  for (unsigned q = 0; q < parts; ++q) sum += sums[q * items + i];
  out[i] = sum;
}

// Rows that are not made of whole aligned 16-byte pieces, or whose distances are not, laid out so that they are: `halves` pieces of `width` elements, each on a
// boundary.  With offsets, the matrices of experts without rows are left out: nobody reads them (85 matrices of 512 x 589, three in use: 8 us; a thread for each piece of all, 32).
struct which_experts {
  const void* offsets;
  bool wide;
  int m;
  __device__ __forceinline__ bool has_rows(size_t e) const { return !offsets || read_offset(offsets, wide, (unsigned)e + 1, m) > read_offset(offsets, wide, (unsigned)e, m); }
};
// The pieces (16 bytes of T, or 8 numbers) of a matrix's halves of rows, 2^spread threads a half: f(row, half, piece) for those of this thread; a matrix for each blockIdx.y.
template <class F> __device__ __forceinline__ void each_piece(size_t rows, unsigned halves, unsigned pieces, unsigned spread, F f) {
  const size_t thread = (size_t)blockIdx.x * 256 + threadIdx.x, lines = rows * halves, step = (size_t)gridDim.x * 256 >> spread;
  for (size_t line = thread >> spread; line < lines; line += step)
    for (unsigned c = (unsigned)thread & ((1u << spread) - 1); c < pieces; c += 1u << spread) f(halves == 2 ? line >> 1 : line, halves == 2 ? (unsigned)line & 1 : 0u, c);
}
template <class T>
__global__ void __launch_bounds__(256) pack_rows_kernel(const T* __restrict__ from, size_t each, size_t outer, size_t stride, unsigned halves, unsigned width, unsigned pieces, unsigned spread,
                                                        which_experts used, T* __restrict__ to) {
  constexpr int V = 16 / sizeof(T);
  if (!used.has_rows(blockIdx.y)) return;
  from += blockIdx.y * outer;
  to += blockIdx.y * each * halves * pieces * V;
  each_piece(each, halves, pieces, spread, [&](size_t row, unsigned h, unsigned piece) {
    const unsigned c = piece * V;
    const T* const f = from + row * stride + (size_t)h * width + c;
    union { T at[V]; uint4 all; } v;
#pragma unroll
    for (int j = 0; j < V; ++j) v.at[j] = c + j < width ? f[j] : from_f32<T>(0.f);
    reinterpret_cast<uint4*>(to)[(row * halves + h) * pieces + piece] = v.all;
  });
}

// The same rows as three planes of 16 bits, [matrix][plane][row][halves][wide], zeros behind a half's width.  A number that is not finite is in the first plane alone.
__global__ void __launch_bounds__(256) split_rows_kernel(const float* __restrict__ from, size_t each, size_t outer, size_t stride, unsigned halves, unsigned width, unsigned pieces, unsigned spread,
                                                         which_experts used, bf16* __restrict__ to) {
  if (!used.has_rows(blockIdx.y)) return;
  from += blockIdx.y * outer;
  const size_t plane = each * halves * pieces;      // in pieces
  to += blockIdx.y * PLANES * plane * 8;
  each_piece(each, halves, pieces, spread, [&](size_t row, unsigned h, unsigned piece) {
    const unsigned c = piece * 8;
    const float* const f = from + row * stride + (size_t)h * width + c;
    float at[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) at[j] = c + j < width ? f[j] : 0.f;
    union { unsigned short at[8]; uint4 all; } v[PLANES];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float x = at[j];
#pragma unroll
      for (int q = 0; q < PLANES; ++q) {
        const unsigned bits = __float_as_uint(x);
        unsigned short r = __bfloat16_as_ushort(__float2bfloat16_rn(x));
        if ((r & 0x7fff) == 0x7f80) r = (unsigned short)(bits >> 16);      // infinity stays, the largest numbers are cut off
        v[q].at[j] = r;
        x = SCALE * (x - __uint_as_float((unsigned)r << 16));      // (both exact)
        if ((bits & 0x7f800000u) == 0x7f800000u) x = 0.f;
      }
    }
#pragma unroll
    for (int q = 0; q < PLANES; ++q) reinterpret_cast<uint4*>(to)[q * plane + (row * halves + h) * pieces + piece] = v[q].all;
  });
}

// dbefore = dout * the activation's slope; gated with out = act(a) b: da = dout b act'(a), db = dout act(a).  Bound by the bytes; a thread asks for two places' pieces before
// it works on either.  98304 bf16 rows of 1024, gated: 156 us with the call (6450 GB/s; one place at a time, and an exponential each for value and slope, 195).
template <class T, int V>
__global__ void __launch_bounds__(256) activation_grad_kernel(const T* __restrict__ dout, size_t stride, const T* __restrict__ before, size_t n, unsigned pieces, bool gated, int kind,
                                                              T* __restrict__ dbefore) {
  constexpr bool FAST = sizeof(T) == 2;
  constexpr int U = 2;
  const size_t all = n * pieces, width = (size_t)pieces * V, both = gated ? 2 * width : width;
  words<T, V> dw[U], aw[U], bw[U];
  size_t at[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const size_t i = ((size_t)blockIdx.x * U + u) * 256 + threadIdx.x;
    at[u] = ~(size_t)0;
    if (i >= all) continue;
    const size_t row = all <= 0xffffffffull ? (unsigned)i / pieces : i / pieces, c = (i - row * pieces) * V;
    at[u] = row * both + c;
    dw[u] = load_words<T, V>(dout + row * stride + c);
    aw[u] = load_words<T, V>(before + at[u]);
    if (gated) bw[u] = load_words<T, V>(before + at[u] + width);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (at[u] == ~(size_t)0) continue;
    T* const to = dbefore + at[u];
    float d[V], a[V], b[V];
    channels(dw[u], d);
    channels(aw[u], a);
    if (gated) channels(bw[u], b);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const act_slope s = with_slope<FAST>(a[v], kind);
      a[v] = (gated ? d[v] * b[v] : d[v]) * s.slope;
      b[v] = d[v] * s.y;
    }
    store_words<T, V>(to, to_words<T, V>(a));
    if (gated) store_words<T, V>(to + width, to_words<T, V>(b));
  }
}

// ---------------------------------------------------------------------------------------------- calls
using encode_call = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
encode_call encoder() {
  static const encode_call call = []() -> encode_call {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
    return reinterpret_cast<encode_call>(f);
  }();
  return call;
}
// A tensor as the copy engine takes boxes from it, 128 bytes of its innermost axis at a time, swizzled.  apart: in elements, of all axes but the innermost.
struct box_axes { size_t size[5], apart[4]; unsigned box[5]; };
template <class T> bool box_map(CUtensorMap& map, const void* at, const box_axes& x) {
  cuuint64_t dims[5], strides[4];
  cuuint32_t boxes[5], steps[5];
  for (int i = 0; i < 5; ++i) { dims[i] = x.size[i]; boxes[i] = x.box[i]; steps[i] = 1; }
  for (int i = 0; i < 4; ++i) strides[i] = x.size[i + 1] > 1 ? x.apart[i] * 2 : 128;      // (an axis of one may lie anywhere)
  return encoder() && encoder()(&map, std::is_same<T, f16>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(at), dims, strides, boxes, steps,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Matrices of `rows` rows of `width` elements, in boxes of 64 (split: `chunks` times 64) neighbours by `box` rows.  Split only where rows are made of whole chunks: otherwise the last
// would go on into the next row.
box_axes plain_axes(size_t width, size_t rows, size_t stride, size_t count, size_t outer, unsigned box, bool split, unsigned chunks) {
  return {{split ? 64 : width, rows, split ? width / 64 : 1, 1, count}, {stride, 64, 0, outer}, {64, box, split ? chunks : 1, 1, 1}};
}

// Matrices as a kernel is given them: as they lie, or packed into the workspace.
struct matrices {
  const void* at;
  size_t width, rows, stride, count, outer;      // count 0: one matrix
  unsigned halves;                               // of the width, each on a boundary of 16 bytes
  size_t bytes;                                  // of an element
  bool split;                                    // to be laid out as planes
  size_t pieces() const { return (half() * bytes + 15) / 16; }
  size_t wide() const { return (half() + 63) / 64 * 64; }      // of a half in a plane
  bool fits() const { return !split && ((reinterpret_cast<uintptr_t>(at) | stride * bytes | (count > 1 ? outer * bytes : 0) | (halves > 1 ? half() * bytes : 0)) & 15) == 0; }
  size_t half() const { return width / halves; }
  size_t all_rows() const { return rows * (count ? count : 1); }
  size_t packed_bytes() const { return fits() ? 0 : tb200::align_up(all_rows() * halves * (split ? PLANES * wide() * 2 : pieces() * 16), 256); }
};
// into `room`, which is moved on; nothing where they fit
template <class T> cudaError_t pack(matrices& x, char*& room, which_experts used, cudaStream_t stream) {
  if (x.fits() || x.width == 0 || x.all_rows() == 0) return cudaSuccess;
  const size_t bytes = x.packed_bytes(), many = x.count ? x.count : 1, pieces = x.split ? x.wide() / 8 : x.pieces();
  const unsigned spread = spread_of(pieces, 5);
  // as many CTAs as can run twice over, all matrices together
  const size_t want = ((x.rows * x.halves << spread) + 255) / 256, most = ((size_t)tb200::current_device_info().sm_count * 16 + many - 1) / many;
  const dim3 grid((unsigned)(want < most ? want : most), (unsigned)many);
  if (x.split) {
    if constexpr (sizeof(T) == 4)
      split_rows_kernel<<<grid, 256, 0, stream>>>(static_cast<const float*>(x.at), x.rows, x.outer, x.stride, x.halves, (unsigned)x.half(), (unsigned)pieces, spread, used,
                                                  reinterpret_cast<bf16*>(room));
    x.width = x.stride = x.halves * x.wide();
    x.count = many * PLANES;
    x.bytes = 2;
    x.split = false;
  } else {
    pack_rows_kernel<T><<<grid, 256, 0, stream>>>(static_cast<const T*>(x.at), x.rows, x.outer, x.stride, x.halves, (unsigned)x.half(), (unsigned)pieces, spread, used, reinterpret_cast<T*>(room));
    x.width = x.stride = x.halves * pieces * 16 / sizeof(T);
  }
  x.at = room;
  x.outer = x.rows * x.stride;
  room += bytes;
  return cudaGetLastError();
}

// How many CTAs: as many as can run, or as there can be tiles
unsigned product_grid(size_t tiles, unsigned a_sm) {
  const size_t most = (size_t)tb200::current_device_info().sm_count * a_sm;
  return (unsigned)(tiles < most ? (tiles ? tiles : 1) : most);
}
size_t most_row_tiles(size_t m, size_t experts, size_t tall) { return m / tall + (m < experts ? m : experts); }

template <class T, class O, int MODE, bool PAIR, bool GATED, int BN, int STAGES>
cudaError_t launch_tc(const CUtensorMap& a, const CUtensorMap& b, const product_plan<T>& p, cudaStream_t stream) {
  using Warps = tc_warps<MODE, O, PAIR>;
  using Shared = tc_shared<PAIR, Warps::WRITERS, BN, STAGES>;
  constexpr size_t CTAS = PAIR ? 2 : 1, WIDE = (GATED ? 64 : 128) * CTAS;
  auto kernel = expert_product_kernel<T, O, MODE, PAIR, GATED, BN, STAGES>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shared::bytes(MOST_EXPERTS));
  if (e != cudaSuccess) return e;
  if constexpr (sizeof(O) == 4) {      // the writers would wait for registers that the CTA does not have
    static thread_local int registers = 0;
    cudaFuncAttributes has;
    if (registers == 0 && cudaFuncGetAttributes(&has, kernel) == cudaSuccess) registers = (has.numRegs + 7) / 8 * 8;
    if (registers * 3 < 2 * WRITERS_REGISTERS + OTHERS_REGISTERS) return cudaErrorInvalidKernelImage;
  }
  const size_t across = ((size_t)p.features + WIDE - 1) / WIDE;
  const size_t tiles = MODE == BY_ROWS ? across * most_row_tiles(p.m, p.experts, BN) : across * (((size_t)p.others + BN - 1) / BN) * p.experts;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(product_grid(tiles * 4 * CTAS, Warps::A_SM) / CTAS * CTAS);      // (four: the parts of a tile)
  cfg.blockDim = dim3(Warps::THREADS);
  cfg.dynamicSmemBytes = Shared::bytes(p.experts);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (PAIR) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = CTAS; attr[n].val.clusterDim.y = 1; attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (!p.first) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, a, b, p);
}

// So few rows an expert that a product is as long as it takes to read the matrices: narrow tiles, and nothing laid out anew that need not be.  Both sides were measured
// with as many rows for each expert; the rule knows the mean alone, and where most rows are a few experts' the wide tiles would take less from fewer rows on.  64 bf16 rows of 2048 for each of
// 64 experts' 2048 outputs, gated: 94 us against 99, 96 rows 122 against 105; of 512 to 512 21 against 25, 27 against 17; 64 32-bit rows of 1024 for 16 experts' 1024 outputs 70
// against 84, 96 rows 97 against 86.
bool few_rows(size_t m, size_t experts) { return m <= 64 * experts; }

template <int MODE, bool A_MN, int BN> cudaError_t launch_fma(const matrices& a, const matrices& b, const product_plan<float>& p, cudaStream_t stream) {
  using Shared = fma_shared<MODE, A_MN, BN>;
  auto kernel = expert_product_f32_kernel<MODE, A_MN, BN>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shared::bytes(MOST_EXPERTS));
  if (e != cudaSuccess) return e;
  const size_t wide = MODE == BY_ROWS && (p.activation & ACT_GATED) ? 64 : 128, across = ((size_t)p.features + wide - 1) / wide;
  const size_t tiles = MODE == BY_ROWS ? across * most_row_tiles(p.m, p.experts, BN) : across * (((size_t)p.others + BN - 1) / BN) * p.experts;
  kernel<<<product_grid(tiles, 3), FMA_THREADS, Shared::bytes(p.experts), stream>>>(static_cast<const float*>(a.at), a.outer, a.stride, static_cast<const float*>(b.at), b.stride, p);
  return cudaGetLastError();
}

// out[i] = rows[i] W[e] (+ the rest) of the expert that row i is of.  w: its matrices' rows are inputs (a_mn: the outputs of an input are neighbours), or outputs.
// Both have been packed.
template <class T> cudaError_t product_by_rows(const matrices& w, const matrices& x, product_plan<T> p, cudaStream_t stream) {
  const bool gated = (p.activation & ACT_GATED) != 0;
  bool few = few_rows(p.m, p.experts);
  p.second = p.a_mn ? (int)(w.halves == 2 ? w.width / 2 : 0) : p.features;
  if constexpr (sizeof(T) == 4) {
    if (p.planes == 1) {
      if (p.a_mn) return few ? launch_fma<BY_ROWS, true, 32>(w, x, p, stream) : launch_fma<BY_ROWS, true, 64>(w, x, p, stream);
      return few ? launch_fma<BY_ROWS, false, 32>(w, x, p, stream) : launch_fma<BY_ROWS, false, 64>(w, x, p, stream);
    }
  }
  cudaError_t e = cudaSuccess;
  const size_t both = (size_t)p.features * (gated ? 2 : 1);
  p.wide_out = in_16_bytes(p.out, p.features, p.features, sizeof(T)) && in_16_bytes(p.before, both, both, sizeof(T));
  p.wide_residual = in_16_bytes(p.residual, p.features, p.residual_stride, sizeof(T));
  p.a_split = w.width % 64 == 0 && !(gated && p.a_mn);
  box_axes of_a = plain_axes(w.width, w.rows, w.stride, w.count, w.outer, 128, p.a_split, 2);
  if (gated && p.a_mn) of_a = {{(size_t)p.features, w.rows, 2, 1, w.count}, {w.stride, (size_t)p.second, 0, w.outer}, {64, 128, 2, 1, 1}};      // 64 of either half
  else if (gated) of_a = {{p.a_split ? 64 : w.width, (size_t)p.features, 2, p.a_split ? w.width / 64 : 1, w.count}, {w.stride, p.features * w.stride, 64, w.outer},
                          {64, 64, 2, p.a_split ? 2u : 1u, 1}};
  for (;; few = true) {      // (again, by single CTAs, if there is no room for pairs)
    p.box = few ? 16 : 128;
    p.b_split = !few && x.width % 64 == 0;
    CUtensorMap a = {}, b = {};
    if (p.k > 0 && (!box_map<T>(a, w.at, of_a) || !box_map<T>(b, x.at, plain_axes(x.width, x.rows, x.stride, p.planes, x.outer, (unsigned)p.box, p.b_split, 2)))) return cudaErrorNotSupported;
    if (few) return gated ? launch_tc<T, T, BY_ROWS, false, true, 64, 2>(a, b, p, stream) : launch_tc<T, T, BY_ROWS, false, false, 64, 2>(a, b, p, stream);
    e = gated ? launch_tc<T, T, BY_ROWS, true, true, 256, 3>(a, b, p, stream) : launch_tc<T, T, BY_ROWS, true, false, 256, 3>(a, b, p, stream);
    if (!tb200::launch_refused(e)) return e;
  }
}

// matrix[e][o][f] = the sum over the expert's rows of others[row][o] features[row][f]
template <class T, class O> cudaError_t product_by_experts(const matrices& features, const matrices& others, product_plan<T> p, cudaStream_t stream) {
  if constexpr (sizeof(T) == 4) {
    if (p.planes == 1) return launch_fma<BY_EXPERTS, true, 64>(features, others, p, stream);
  }
  p.wide_out = in_16_bytes(p.matrix, p.features, p.features, sizeof(O));
  p.a_split = features.width % 64 == 0;
  p.b_split = others.width % 64 == 0;
  CUtensorMap a = {}, b = {};
  if (p.m > 0 && (!box_map<T>(a, features.at, plain_axes(features.width, features.rows, features.stride, p.planes, features.outer, DEEP, p.a_split, 2)) ||
                  !box_map<T>(b, others.at, plain_axes(others.width, others.rows, others.stride, p.planes, others.outer, DEEP, p.b_split, 2))))
    return cudaErrorNotSupported;
  if (p.features > 128) {      // (a pair's tile has 256: of fewer than half of them the second CTA would have nothing)
    const cudaError_t e = launch_tc<T, O, BY_EXPERTS, true, false, 256, 3>(a, b, p, stream);
    if (!tb200::launch_refused(e)) return e;      // (no room for pairs)
  }
  return launch_tc<T, O, BY_EXPERTS, false, false, 128, 3>(a, b, p, stream);
}

// what is laid out anew is read 16 bytes at a time, and by the copy engine
bool on_16_bytes(const void* d_ws) { return (reinterpret_cast<uintptr_t>(d_ws) & 15) == 0; }
bool sizes_fit(size_t n, size_t experts, size_t in, size_t out) { return n <= MOST_ROWS && experts >= 1 && experts <= (size_t)MOST_EXPERTS && in < MOST_CHANNELS && out < MOST_CHANNELS; }
// 32-bit rows go to the tensor cores, as planes, where products are longer than it takes to lay the planes out: not few rows, and 128 or more channels on both sides (256 rows of
// 64 for 16 experts' 64 outputs: 14 us by multiply-adds against 21; 256 of 128 to 2048: 98 against 42).  Sums over very many rows do too, because one
// multiply-add after another rounds them too often.
template <class T> bool in_planes(size_t n, size_t experts, size_t in, size_t out, bool grad) {
  return sizeof(T) == 4 && in && out && !few_rows(n, experts) && ((in >= 128 && out >= 128) || (grad && n >= 2048 * experts));
}
template <class T> void set_planes(product_plan<T>& p, bool split) {
  p.planes = split ? PLANES : 1;
  p.a_planes = split ? A_PLANES : 0;
  p.b_planes = split ? B_PLANES : 0;
}
bool activation_known(int a) { return a == ACT_NONE || (a & ~ACT_GATED) == ACT_SILU || (a & ~ACT_GATED) == ACT_GELU; }
// weight as it lies: an input's outputs are neighbours, or an output's inputs
matrices weights_of(const void* d_weight, size_t experts, size_t in, size_t out, size_t expert_stride, size_t stride, bool inputs_inside, unsigned halves, size_t bytes, bool split) {
  if (inputs_inside) return {d_weight, in, out, stride, experts, expert_stride, 1, bytes, split};
  return {d_weight, out, in, stride, experts, expert_stride, halves, bytes, split};
}
bool weights_fit(size_t experts, size_t in, size_t out, size_t expert_stride, size_t stride, bool inputs_inside) {
  const size_t width = inputs_inside ? in : out, rows = inputs_inside ? out : in;
  return stride >= width && (experts == 1 || expert_stride >= (rows ? (rows - 1) * stride + width : 0));
}
// how many pieces of an expert's rows are added up side by side: as long as a warp has eight rows, enough CTAs for every SM to hold eight
unsigned sum_parts(size_t n, size_t experts, size_t out) {
  const size_t ctas = ((out + 255) / 256) * experts, most = (size_t)tb200::current_device_info().sm_count * 8, rows = n / experts / 64;
  size_t parts = ctas ? (most + ctas - 1) / ctas : 1;
  if (parts > rows) parts = rows;
  return (unsigned)(parts < 1 ? 1 : parts > 256 ? 256 : parts);
}
}  // namespace

TB200_API int tb200_expert_product(const void* d_rows, size_t rows_stride, const void* d_offsets, int offset_t, const void* d_weight, size_t expert_stride, size_t weight_stride,
                                   int inputs_inside, const void* d_bias, const void* d_residual, size_t residual_stride, int activation, size_t n, size_t num_experts, size_t in,
                                   size_t out, int t, void* d_out, void* d_before, void* d_ws, size_t* ws_bytes, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    return by_index_dtype(offset_t, [&](auto iv) -> int {
      const bool gated = (activation & ACT_GATED) != 0;
      if (!sizes_fit(n, num_experts, in, out) || !activation_known(activation) || (gated && out % 2) || !on_16_bytes(d_ws)) return ERR_INVALID;
      const size_t width = gated ? out / 2 : out;
      const bool split = in_planes<T>(n, num_experts, in, out, false);
      matrices w = weights_of(d_weight, num_experts, in, out, expert_stride, weight_stride, inputs_inside != 0, gated ? 2 : 1, sizeof(T), split), x = {d_rows, in, n, rows_stride, 0, 0, 1, sizeof(T), split};
      int rc;
      if (workspace_gate(d_ws, ws_bytes, sizeof(tb200::ws_header) + w.packed_bytes() + x.packed_bytes(), rc)) return rc;
      if (n == 0 || width == 0) return 0;
      if (!d_offsets || !d_out || (in && (!d_rows || !d_weight)) || rows_stride < in || (d_residual && residual_stride < width) ||
          !weights_fit(num_experts, in, out, expert_stride, weight_stride, inputs_inside != 0))
        return ERR_INVALID;
      product_plan<T> p = {};
      p.offsets = d_offsets;
      p.wide = sizeof(iv) == 8;
      p.experts = (unsigned)num_experts;
      p.m = (int)n;
      p.k = (int)in;
      p.features = (int)width;
      p.a_mn = !inputs_inside;
      p.bias = static_cast<const T*>(d_bias);
      p.residual = static_cast<const T*>(d_residual);
      p.residual_stride = residual_stride;
      p.out = static_cast<T*>(d_out);
      p.before = static_cast<T*>(d_before);
      p.activation = activation;
      p.first = true;
      p.hdr = static_cast<tb200::ws_header*>(d_ws);
      set_planes(p, split);
      char* room = static_cast<char*>(d_ws) + sizeof(tb200::ws_header);
      cudaError_t e = pack<T>(w, room, {d_offsets, p.wide, p.m}, stream);
      if (e == cudaSuccess) e = pack<T>(x, room, {}, stream);
      return (int)(e == cudaSuccess ? product_by_rows<T>(w, x, p, stream) : e);
    });
  });
}

TB200_API int tb200_expert_product_grad(const void* d_dout, size_t dout_stride, const void* d_rows, size_t rows_stride, const void* d_offsets, int offset_t, const void* d_weight,
                                        size_t expert_stride, size_t weight_stride, int inputs_inside, size_t n, size_t num_experts, size_t in, size_t out, int t, int grad_t,
                                        int accumulate, void* d_drows, void* d_dweight, float* d_dbias, void* d_ws, size_t* ws_bytes, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    if (grad_t != t && grad_t != TB200_F32) return ERR_UNSUPPORTED;
    return by_index_dtype(offset_t, [&](auto iv) -> int {
      if (!sizes_fit(n, num_experts, in, out) || !on_16_bytes(d_ws)) return ERR_INVALID;
      const bool split = in_planes<T>(n, num_experts, in, out, true);
      matrices w = weights_of(d_weight, num_experts, in, out, expert_stride, weight_stride, inputs_inside != 0, 1, sizeof(T), split), x = {d_rows, in, n, rows_stride, 0, 0, 1, sizeof(T), split},
               d = {d_dout, out, n, dout_stride, 0, 0, 1, sizeof(T), split};
      const unsigned parts = d_dbias ? sum_parts(n, num_experts, out) : 1;
      const size_t sums = parts > 1 ? tb200::align_up((size_t)parts * num_experts * out * 4, 256) : 0;
      const bool products = n && in && out;      // otherwise what is left are zeros and the gradient of bias, and no product reads an operand (they may be NULL)
      int rc;
      if (workspace_gate(d_ws, ws_bytes, sizeof(tb200::ws_header) + sums + (products ? w.packed_bytes() + x.packed_bytes() + d.packed_bytes() : 0), rc)) return rc;
      if (out == 0 && (n == 0 || in == 0)) return 0;
      if (!d_offsets || (in && n && (!d_drows || (out && (!d_rows || !d_weight)))) || (in && out && !d_dweight) || (out && n && !d_dout) || rows_stride < in || dout_stride < out ||
          !weights_fit(num_experts, in, out, expert_stride, weight_stride, inputs_inside != 0))
        return ERR_INVALID;
      char* room = static_cast<char*>(d_ws) + sizeof(tb200::ws_header);
      float* const partial = reinterpret_cast<float*>(room);
      room += sums;
      cudaError_t e = cudaSuccess;
      if (products) {
        e = pack<T>(w, room, {d_offsets, sizeof(iv) == 8, (int)n}, stream);
        if (e == cudaSuccess) e = pack<T>(x, room, {}, stream);
        if (e == cudaSuccess) e = pack<T>(d, room, {}, stream);
        if (e != cudaSuccess) return (int)e;
      }
      product_plan<T> p = {};
      p.offsets = d_offsets;
      p.wide = sizeof(iv) == 8;
      p.experts = (unsigned)num_experts;
      p.m = (int)n;
      p.hdr = static_cast<tb200::ws_header*>(d_ws);
      p.first = true;
      set_planes(p, split);
      if (n && in) {
        product_plan<T> q = p;
        q.k = (int)out;
        q.features = (int)in;
        q.a_mn = inputs_inside != 0;
        q.out = static_cast<T*>(d_drows);
        e = product_by_rows<T>(w, d, q, stream);
        if (e != cudaSuccess) return (int)e;
        p.first = false;
      }
      if (in && out) {
        const matrices &inside = inputs_inside ? x : d, &around = inputs_inside ? d : x;
        p.features = (int)(inputs_inside ? in : out);
        p.others = (int)(inputs_inside ? out : in);
        p.matrix = d_dweight;
        p.accumulate = accumulate != 0;
        e = grad_t == t ? product_by_experts<T, T>(inside, around, p, stream) : product_by_experts<T, float>(inside, around, p, stream);
        if (e != cudaSuccess) return (int)e;
      }
      if (d_dbias && out) {
        float* const to = parts > 1 ? partial : d_dbias;
        auto add = [&](auto vv) {
          constexpr int V = decltype(vv)::value;
          cudaLaunchConfig_t cfg = {};
          cfg.gridDim = dim3((unsigned)((out + 32 * V - 1) / (32 * V)), (unsigned)num_experts, parts);
          cfg.blockDim = dim3(SUM_BLOCK);
          cfg.stream = stream;
          cudaLaunchAttribute attr[1];
          attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
          attr[0].val.programmaticStreamSerializationAllowed = 1;
          cfg.attrs = attr;
          cfg.numAttrs = in ? 1 : 0;      // beside the products: they are this call's, so what dout comes from is done
          return cudaLaunchKernelEx(&cfg, row_sums_kernel<T, V>, static_cast<const T*>(d_dout), dout_stride, d_offsets, sizeof(iv) == 8, (unsigned)num_experts, (int)n, (int)out, to,
                                    in ? nullptr : p.hdr);
        };
        e = in_16_bytes(d_dout, out, dout_stride, sizeof(T)) ? add(std::integral_constant<int, 16 / sizeof(T)>()) : add(std::integral_constant<int, 1>());
        if (e == cudaSuccess && parts > 1)
          e = tb200::launch_after(join_sums_kernel, (num_experts * out + SUM_BLOCK - 1) / SUM_BLOCK, SUM_BLOCK, 0, stream, partial, num_experts * out, parts, d_dbias);
      }
      return (int)e;
    });
  });
}

TB200_API int tb200_expert_activation_grad(const void* d_dout, size_t dout_stride, const void* d_before, int activation, size_t n, size_t width, int t, void* d_dbefore,
                                           tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    const bool gated = (activation & ACT_GATED) != 0;
    if (!activation_known(activation) || activation == ACT_NONE || n > MOST_ROWS || width >= MOST_CHANNELS) return ERR_INVALID;
    if (n == 0 || width == 0) return 0;
    if (!d_dout || !d_before || !d_dbefore || dout_stride < width) return ERR_INVALID;
    auto go = [&](auto vv) -> int {
      constexpr int V = decltype(vv)::value;
      const size_t grid = (n * (width / V) + 511) / 512;
      if (grid > 0x7fffffffull) return ERR_INVALID;
      activation_grad_kernel<T, V><<<(unsigned)grid, 256, 0, stream>>>(static_cast<const T*>(d_dout), dout_stride, static_cast<const T*>(d_before), n, (unsigned)(width / V), gated,
                                                                      activation & ~ACT_GATED, static_cast<T*>(d_dbefore));
      return (int)cudaGetLastError();
    };
    if (in_16_bytes(d_dout, width, dout_stride, sizeof(T)) && in_16_bytes(d_before, width, width, sizeof(T)) && in_16_bytes(d_dbefore, width, width, sizeof(T)))
      return go(std::integral_constant<int, 16 / sizeof(T)>());
    return go(std::integral_constant<int, 1>());
  });
}
