// C ABI: tb200_expert_route and tb200_expert_route_grad.
#include "abi_rows.cuh"

using namespace tb200_abi;
using namespace tb200_rows;

namespace {
constexpr int MOST_EXPERTS = 1024, MOST_CHOICES = 32, MOST_GROUPS = 32;
constexpr int BLOCK = 128;
constexpr unsigned ALL = tb200::FULL_MASK;

struct route_plan {
  const float* bias;      // may be NULL
  unsigned experts, choices, groups, group_choices, group_best;
  bool sigmoid, renormalize;
  float scale;
};
// the logits' order is the scores', and no scores are added up
__device__ __forceinline__ bool exact_by_logits(const route_plan& p) { return !p.bias && !(p.groups > 1 && p.group_best > 1); }

// Up to 32 / L tokens a warp, L neighbouring lanes each; lane l of them has experts l * PER to l * PER + PER - 1.
template <int L> __device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
  return x;
}
template <int L> __device__ __forceinline__ double lanes_sum(double x) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
  return x;
}
template <int L> __device__ __forceinline__ unsigned lanes_max(unsigned x) {
  if constexpr (L == 32) {
    return __reduce_max_sync(ALL, x);
  } else {
#pragma unroll
    for (int o = L / 2; o; o >>= 1) { const unsigned y = __shfl_xor_sync(ALL, x, o); x = y > x ? y : x; }
    return x;
  }
}
template <int L> __device__ __forceinline__ unsigned long long lanes_max(unsigned long long x) {
#pragma unroll
  for (int o = L / 2; o; o >>= 1) { const unsigned long long y = __shfl_xor_sync(ALL, x, o); x = y > x ? y : x; }
  return x;
}

// Numbers (no NaN, no -0) as integers in the same order, above 0, which stands for an expert that is not open.  FAST: functions good to a few 2^-22 and, of the
// exponential's argument x, 2^-24 |x|.
template <class R> struct ordered;
template <> struct ordered<float> {
  using key = unsigned;
  static __device__ __forceinline__ key of(float x) { const unsigned u = __float_as_uint(x); return u & 0x80000000u ? ~u : u | 0x80000000u; }
  static __device__ __forceinline__ float value(key k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
  static __device__ __forceinline__ float exp_of(float x) { return __expf(x); }
  static __device__ __forceinline__ float over(float a, float b) { return __fdividef(a, b); }
};
template <> struct ordered<double> {
  using key = unsigned long long;
  static __device__ __forceinline__ key of(double x) { const unsigned long long u = (unsigned long long)__double_as_longlong(x); return u >> 63 ? ~u : u | 1ull << 63; }
  static __device__ __forceinline__ double value(key k) { return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k)); }
  static __device__ __forceinline__ double exp_of(double x) { return exp(x); }
  static __device__ __forceinline__ double over(double a, double b) { return a / b; }
};

// the best of a lane's own experts in [low, high) other than `but`, the first of equal ones
template <class K, int PER> __device__ __forceinline__ K best_of(const K (&order)[PER], int first, int low, int high, int but, int& at) {
  K best = 0;
  at = -1;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (order[i] > best && first + i >= low && first + i < high && first + i != but) { best = order[i]; at = first + i; }
  return best;
}
template <class K> struct two { K first, second; };      // the best two of some
template <class K> __device__ __forceinline__ two<K> both_of(two<K> a, two<K> b) {
  const K less = a.first < b.first ? a.first : b.first, second = a.second > b.second ? a.second : b.second;
  return {a.first > b.first ? a.first : b.first, less > second ? less : second};
}

// The choices of a token, choice c in its lane c (-1: none).
//
// Scores are compared as 64-bit numbers would be.  Where the order is the logits' (no bias, and no sums of scores of groups) it is exact as it is.
// Otherwise the scores are 32-bit numbers that are off by up to `slack`: two neighbours in the order that are nearer than that, and the last group
// kept and the first left out, are `unsure`, and the token is done again in 64 bits.  (Equal logits with equal biases are as equal there.)
template <class R, int L, int PER, class T> __device__ __forceinline__ bool choose(const route_plan& p, const T* row, bool whole, uint2* candidates, int& chosen) {
  using O = ordered<R>;
  using K = typename O::key;
  const int lane = threadIdx.x % L, first = lane * PER, experts = (int)p.experts;
  const bool sums = p.groups > 1 && p.group_best > 1, exact = sizeof(R) == 8 || (!p.bias && !sums);
  R x[PER];      // logits; -inf: not open
  if (whole) {   // rows of whole 16-byte pieces, all of them experts
    constexpr int V = 16 / sizeof(T) < PER ? 16 / sizeof(T) : PER;
#pragma unroll
    for (int i = 0; i < PER; i += V) {
      float f[V];
      channels(load_words<T, V>(row + first + i), f);
#pragma unroll
      for (int v = 0; v < V; ++v) x[i + v] = f[v] > -INFINITY ? (R)f[v] : -(R)INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float f = first + i < experts ? to_f32(row[first + i]) : -INFINITY;
      x[i] = f > -INFINITY ? (R)f : -(R)INFINITY;
    }
  }
  auto key_of = [&](R v) { return v > -(R)INFINITY ? O::of(v + (R)0) : (K)0; };      // neither NaN nor -0
  // of the softmax: the largest logit, and the sum of exp(logit - largest); an infinite logit leaves the others nothing
  R top = 0, sum = 1;
  auto share = [&](R v) { return v == top ? (R)1 : O::exp_of(v - top); };
  if (!p.sigmoid && !exact_by_logits(p)) {
    R mine = x[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) mine = x[i] > mine ? x[i] : mine;
    const K best = lanes_max<L>(key_of(mine));
    if (best) top = O::value(best);
    R own = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) own += x[i] > -(R)INFINITY ? share(x[i]) : (R)0;
    sum = lanes_sum<L>(own);
    if (!best) sum = 1;
  }
  const R under = (R)1 / sum;
  auto score_of = [&](R v) { return p.sigmoid ? O::over((R)1, (R)1 + O::exp_of(-v)) : share(v) * under; };
  auto score = [&](K k) { return score_of(O::value(k)); };
  if (p.bias) {
    R bias[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) bias[i] = first + i < experts ? (R)p.bias[first + i] : (R)0;
    if (p.sigmoid) {
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = x[i] > -(R)INFINITY ? O::over((R)1, (R)1 + O::exp_of(-x[i])) + bias[i] : x[i];
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = x[i] > -(R)INFINITY ? share(x[i]) * under + bias[i] : x[i];
    }
  }
  K order[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) order[i] = key_of(x[i]);
  // exponentials of rounded differences, sums of up to 1024 of them: good to 2^-18 of the largest score; a sum with a bias to 2^-24 of itself
  const R largest = p.sigmoid ? (R)1 : under;
  auto slack = [&](R v) { return (R)0x1p-18 * largest + (R)0x1p-22 * (v < 0 ? -v : v); };
  bool unsure = false;
  if (p.groups > 1) {
    const int size = experts / (int)p.groups, across = size / PER;
    auto rank_of = [&](two<K> b) {      // what a group counts: the key of the sum, or of its best
      if (!sums || !b.first) return b.first;
      const R x = p.bias ? O::value(b.first) : score(b.first), y = !b.second ? (R)0 : p.bias ? O::value(b.second) : score(b.second);
      return O::of(x + y + (R)0);
    };
    K mine = 0;                 // of the group whose number is `own`
    int own, stride;            // group g's is known to lane g * stride
    const bool aligned = size % PER == 0 && (across & (across - 1)) == 0;
    if (aligned) {              // a lane's experts are of one group, the lanes of a group a power of two
      two<K> b = {0, 0};
#pragma unroll
      for (int i = 0; i < PER; ++i) b = both_of(b, two<K>{order[i], 0});
#pragma unroll
      for (int o = 1; o < L; o <<= 1) {
        const two<K> other = {__shfl_xor_sync(ALL, b.first, o), __shfl_xor_sync(ALL, b.second, o)};
        if (o < across) b = both_of(b, other);
      }
      mine = rank_of(b);
      own = lane / across;
      stride = across;
      if (own >= (int)p.groups) mine = 0;
    } else {
      own = lane;
      stride = 1;
      for (int g = 0; g < (int)p.groups; ++g) {
        two<K> b;
        int at;
        const K one = best_of(order, first, g * size, (g + 1) * size, -1, at);
        b.first = lanes_max<L>(one);
        // the lowest lane that has it gives up that one expert
        const unsigned having = __ballot_sync(ALL, one == b.first) >> (threadIdx.x % 32 / L * L) & (L == 32 ? ~0u : (1u << L % 32) - 1);
        const K two_ = best_of(order, first, g * size, (g + 1) * size, __ffs(having) - 1 == lane ? at : -1, at);
        b.second = lanes_max<L>(two_);
        const K r = rank_of(b);
        if (lane == g) mine = r;
      }
    }
    int before = 0;
    for (int g = 0; g < (int)p.groups; ++g) {
      const K other = __shfl_sync(ALL, mine, g * stride, L);
      before += other > mine || (other == mine && g < own);
    }
    const bool stays = own < (int)p.groups && before < (int)p.group_choices;
    if (!exact) {
      const K last = ~lanes_max<L>(stays ? ~mine : (K)0), next = lanes_max<L>(stays ? (K)0 : mine);
      if (next && O::value(last) - O::value(next) < 2 * slack(O::value(last))) unsure = true;
    }
    if (aligned) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (!stays) order[i] = 0;
    } else {
      const unsigned kept = __ballot_sync(ALL, stays) >> (threadIdx.x % 32 / L * L);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (first + i < experts && !(kept >> ((first + i) / size) & 1)) order[i] = 0;
    }
  }
  chosen = -1;
  // A whole warp sorts its lanes' best.  What is no worse than the last of those that are asked for, a few more than those, are the candidates; they are sorted, one a lane.
  if constexpr (L == 32 && sizeof(R) == 4) {
    const int asked = (int)p.choices + (exact ? 0 : 1);
    if (asked <= 32) {
      K mine = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) mine = order[i] > mine ? order[i] : mine;
      K sorted = mine;
#pragma unroll
      for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size / 2; o; o >>= 1) {
          const K other = __shfl_xor_sync(ALL, sorted, o);
          const bool larger = ((lane & size) == 0) == ((lane & o) == 0);      // of the two, this lane keeps the larger
          sorted = (other > sorted) == larger ? other : sorted;
        }
      K least = __shfl_sync(ALL, sorted, asked - 1);
      least = least ? least : 1;
      const unsigned below = (1u << lane) - 1;
      int count = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const bool is = order[i] >= least;
        const unsigned these = __ballot_sync(ALL, is);
        const int at = count + __popc(these & below);
        if (is && at < 32) candidates[at] = make_uint2(order[i], (unsigned)(first + i));
        count += __popc(these);
      }
      __syncwarp();
      if (count <= 32) {
        const uint2 c = lane < count ? candidates[lane] : make_uint2(0, 0xffffffffu);
        K key = c.x;
        unsigned at = c.y;
#pragma unroll
        for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
          for (int o = size / 2; o; o >>= 1) {
            const K other = __shfl_xor_sync(ALL, key, o);
            const unsigned other_at = __shfl_xor_sync(ALL, at, o);
            const bool larger = ((lane & size) == 0) == ((lane & o) == 0);
            if ((other > key || (other == key && other_at < at)) == larger) { key = other; at = other_at; }
          }
        if (lane < (int)p.choices && key) chosen = (int)at;
        const K next = __shfl_down_sync(ALL, key, 1);
        const unsigned next_at = __shfl_down_sync(ALL, at, 1);
        if (!exact && lane < (int)p.choices && lane < 31 && next && O::value(key) - O::value(next) < slack(O::value(key))) {
          const float u = to_f32(row[at]), v = to_f32(row[next_at]);
          unsure |= !(u == v && (!p.bias || p.bias[at] == p.bias[next_at]));
        }
        return unsure;
      }
    }
  }
  K last = 0, mine = 0;
  int last_at = -1, own_at = -1;      // own_at: which of this lane's experts is its best
  auto best = [&] {
    mine = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (order[i] > mine) { mine = order[i]; own_at = i; }
  };
  best();
  const unsigned segment = threadIdx.x % 32 / L * L, all_lanes = L == 32 ? ~0u : (1u << L % 32) - 1;
  for (int c = 0; c < (int)p.choices + (exact ? 0 : 1); ++c) {
    const K next = lanes_max<L>(mine);
    const int winner = __ffs(__ballot_sync(ALL, mine == next) >> segment & all_lanes) - 1, next_at = __shfl_sync(ALL, first + own_at, winner, L);
    if (!exact && c > 0 && next && O::value(last) - O::value(next) < slack(O::value(last))) {
      const float x = to_f32(row[last_at]), y = to_f32(row[next_at]);
      unsure |= !(x == y && (!p.bias || p.bias[last_at] == p.bias[next_at]));
    }
    if (next && lane == c && c < (int)p.choices) chosen = next_at;
    const int taken = lane == winner ? own_at : -1;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i == taken) order[i] = 0;
    best();
    last = next;
    last_at = next_at;
  }
  return unsure;
}
// (not inlined: few tokens come here, and its registers would be all tokens')
template <int L, int PER, class T> __device__ __noinline__ int choose_in_64(const route_plan& p, const T* row, bool whole) {
  int chosen;
  choose<double, L, PER>(p, row, whole, nullptr, chosen);
  return chosen;
}

// Of the softmax over a row's open experts: its largest logit and the sum of exp(logit - largest).
struct softmax_of {
  float top, sum;
  __device__ __forceinline__ float share(float x) const { return x == top ? 1.f : expf(x - top); }      // times the sum
};
template <int L> __device__ __forceinline__ float lanes_max_of(float x) { return ordered<float>::value(lanes_max<L>(ordered<float>::of(x + 0.f))); }
template <int L, int V, class T> __device__ __forceinline__ softmax_of softmax_over(const T* row, unsigned pieces) {
  const unsigned lane = threadIdx.x % L;
  softmax_of all;
  float top = -INFINITY, sum = 0.f;
  for (unsigned c = lane; c < pieces; c += L) {
    float f[V];
    channels(load_words<T, V>(row + c * V), f);
#pragma unroll
    for (int v = 0; v < V; ++v) top = f[v] > top ? f[v] : top;
  }
  all.top = lanes_max_of<L>(top);
  for (unsigned c = lane; c < pieces; c += L) {
    float f[V];
    channels(load_words<T, V>(row + c * V), f);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (f[v] > -INFINITY) sum += all.share(f[v]);
  }
  all.sum = lanes_sum<L>(sum);
  return all;
}

// w = score (/ the sum of the chosen ones' scores) of the chosen expert's logit x.  Quotients are made of exponentials relative to the largest, so that
// they hold where the scores themselves vanish: with c = min(largest, 0), sigmoid(x) e^-c = e^(x - c) / (1 + e^x) for x <= 0.
struct weight_of { float w, other; };      // the quotient or the score; 1 - sigmoid(x)
template <int L> __device__ __forceinline__ weight_of weigh(bool chosen, float x, bool sigmoid, bool renormalize, const softmax_of& all) {
  weight_of r = {0.f, 0.f};
  if (sigmoid) {
    const float e = expf(-fabsf(x));
    r.other = x >= 0.f ? e / (1.f + e) : 1.f / (1.f + e);
    if (!renormalize) {
      r.w = x >= 0.f ? 1.f / (1.f + e) : e / (1.f + e);
    } else {
      const float c = fminf(lanes_max_of<L>(chosen ? x : -INFINITY), 0.f);
      r.w = x > 0.f ? 1.f / (1.f + e) : (x == c ? 1.f : expf(x - c)) / (1.f + e);
    }
  } else if (renormalize) {
    const softmax_of some = {lanes_max_of<L>(chosen ? x : -INFINITY), 1.f};
    r.w = some.share(x);
  } else {
    r.w = all.share(x) / all.sum;
  }
  if (!chosen) r.w = 0.f;
  if (renormalize) {
    const float sum = lanes_sum<L>(r.w);
    r.w = sum > 0.f ? r.w / sum : 0.f;
  }
  return r;
}

// Bound by instructions, 1120 for a token of 256 experts in eight groups: 16384 of them take 30 us, 25 without the 35 that are done again in 64 bits and end last
// (chosen one after another 39; a warp's lanes with every 32nd expert, groups one after another, 71).  48 tokens take 5 us, the call 11.
template <class T, int L, int PER>
__global__ void __launch_bounds__(BLOCK) expert_route_kernel(const T* __restrict__ logits, size_t stride, unsigned n, route_plan p, bool whole, int* __restrict__ experts,
                                                           float* __restrict__ weights) {
  const unsigned place = blockIdx.x * (BLOCK / L) + threadIdx.x / L, token = place < n ? place : n - 1, lane = threadIdx.x % L;
  const T* const row = logits + token * stride;
  __shared__ uint2 candidates[L == 32 ? BLOCK : 1];
  int chosen;
  const bool unsure = choose<float, L, PER>(p, row, whole, candidates + (L == 32 ? threadIdx.x / 32 * 32 : 0), chosen);
  if (__any_sync(ALL, unsure)) chosen = choose_in_64<L, PER>(p, row, whole);
  softmax_of all = {0.f, 1.f};
  constexpr unsigned V = 16 / sizeof(T);
  if (!p.sigmoid && !p.renormalize) all = whole ? softmax_over<L, V>(row, p.experts / V) : softmax_over<L, 1>(row, p.experts);
  const float x = chosen >= 0 ? to_f32(row[chosen]) : 0.f;
  const weight_of r = weigh<L>(chosen >= 0, x, p.sigmoid, p.renormalize, all);
  if (place < n && lane < p.choices) {
    experts[(size_t)token * p.choices + lane] = chosen;
    weights[(size_t)token * p.choices + lane] = p.scale * r.w;
  }
}

// L lanes a token: what every expert's logit gets (zero but for the whole softmax), then the chosen ones' in their places.
//   renormalised: w_c (g_c - sum of g w) (sigmoid: times 1 - s_c);   softmax: p_e (G_e - sum of g p);   sigmoid: g_c s_c (1 - s_c),
// with G_e the sum of g over the choices of e.  Bound by the launch: 16384 tokens of 64 experts take 8 us (a warp a token
// 16.5), of which 0.8 are bytes.
template <class T, int L, int V, bool DENSE>
__global__ void __launch_bounds__(BLOCK) expert_route_grad_kernel(const float* __restrict__ dweights, const int* __restrict__ ids, const T* __restrict__ logits, size_t stride, unsigned n,
                                                                route_plan p, T* __restrict__ dlogits) {
  const unsigned place = blockIdx.x * (BLOCK / L) + threadIdx.x / L, token = place < n ? place : n - 1, lane = threadIdx.x % L;
  const T* const row = logits + token * stride;
  T* const to = dlogits + (size_t)token * p.experts;
  const unsigned pieces = p.experts / V;
  const int id = lane < p.choices ? ids[(size_t)token * p.choices + lane] : -1;
  float x = (unsigned)id < p.experts ? to_f32(row[id]) : -INFINITY;
  const bool chosen = x > -INFINITY;
  x = chosen ? x : 0.f;
  const float g = chosen ? p.scale * dweights[(size_t)token * p.choices + lane] : 0.f;
  softmax_of all = {0.f, 1.f};
  if (DENSE) all = softmax_over<L, V>(row, pieces);
  const weight_of r = weigh<L>(chosen, x, p.sigmoid, p.renormalize, all);
  const float mean = p.renormalize || DENSE ? lanes_sum<L>(g * r.w) : 0.f;
  // of this choice; choices of the same expert are added up, in their order
  const float own = DENSE ? g : p.renormalize ? r.w * (g - mean) * (p.sigmoid ? r.other : 1.f) : g * r.w * r.other;
  float d = 0.f;
  for (unsigned c = 0; c < p.choices; ++c) {
    const int other = __shfl_sync(ALL, chosen ? id : -1, c, L);
    const float add = __shfl_sync(ALL, own, c, L);
    if (other == id) d += add;
  }
  if (DENSE) d = r.w * (d - mean);
  if (place < n)
    for (unsigned c = lane; c < pieces; c += L) {
      float f[V];
      if (DENSE) channels(load_words<T, V>(row + c * V), f);
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = DENSE && f[v] > -INFINITY ? -(all.share(f[v]) / all.sum) * mean : 0.f;
      store_words<T, V>(to + c * V, to_words<T, V>(f));
    }
  __syncwarp();
  if (chosen && place < n) to[id] = from_f32<T>(d);
}

// (lanes a token, experts a lane) for so many experts, and `held` choices or groups, one a lane: as few lanes as leave each about eight experts
template <class F> int by_lanes(size_t experts, size_t held, F f) {
  using std::integral_constant;
  if (experts <= 32 && held <= 8) return f(integral_constant<int, 8>(), integral_constant<int, 4>());
  if (experts <= 64 && held <= 8) return f(integral_constant<int, 8>(), integral_constant<int, 8>());
  if (experts <= 128 && held <= 16) return f(integral_constant<int, 16>(), integral_constant<int, 8>());
  if (experts <= 256) return f(integral_constant<int, 32>(), integral_constant<int, 8>());
  if (experts <= 512) return f(integral_constant<int, 32>(), integral_constant<int, 16>());
  return f(integral_constant<int, 32>(), integral_constant<int, 32>());
}
bool sizes_fit(size_t n, size_t experts, size_t choices) {
  return experts >= 1 && experts <= (size_t)MOST_EXPERTS && choices >= 1 && choices <= (size_t)MOST_CHOICES && choices <= experts && n <= 0x3fffffffull / choices;
}
}  // namespace

TB200_API int tb200_expert_route(const void* d_logits, size_t logits_stride, size_t n, size_t num_experts, int t, const float* d_bias, size_t choices, int scores, size_t groups,
                                 size_t group_choices, int group_best, int renormalize, float scale, int* d_experts, float* d_weights, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    if (!sizes_fit(n, num_experts, choices) || (scores != TB200_SOFTMAX && scores != TB200_SIGMOID) || groups < 1 || groups > (size_t)MOST_GROUPS || num_experts % groups ||
        group_choices < 1 || group_choices > groups || (group_best != 1 && group_best != 2))
      return ERR_INVALID;
    if (n == 0) return 0;
    if (!d_logits || !d_experts || !d_weights || logits_stride < num_experts) return ERR_INVALID;
    route_plan p = {d_bias, (unsigned)num_experts, (unsigned)choices, (unsigned)groups, (unsigned)group_choices, (unsigned)group_best, scores == TB200_SIGMOID, renormalize != 0, scale};
    if (group_choices == groups) p.groups = 1;      // all of them stay
    return by_lanes(num_experts, choices > p.groups ? choices : p.groups, [&](auto lanes, auto per) -> int {
      constexpr int L = decltype(lanes)::value, PER = decltype(per)::value, TOKENS = BLOCK / L;
      const bool whole = num_experts == (size_t)L * PER && in_16_bytes(d_logits, num_experts, logits_stride, sizeof(T));
      expert_route_kernel<T, L, PER><<<(unsigned)((n + TOKENS - 1) / TOKENS), BLOCK, 0, stream>>>(static_cast<const T*>(d_logits), logits_stride, (unsigned)n, p, whole, d_experts, d_weights);
      return (int)cudaGetLastError();
    });
  });
}

TB200_API int tb200_expert_route_grad(const float* d_dweights, const int* d_experts, const void* d_logits, size_t logits_stride, size_t n, size_t num_experts, size_t choices, int t,
                                      int scores, int renormalize, float scale, void* d_dlogits, tb200_stream_t stream) {
  return by_row_dtype(t, [&](auto tv) -> int {
    using T = decltype(tv);
    if (!sizes_fit(n, num_experts, choices) || (scores != TB200_SOFTMAX && scores != TB200_SIGMOID)) return ERR_INVALID;
    if (n == 0) return 0;
    if (!d_dweights || !d_experts || !d_logits || !d_dlogits || logits_stride < num_experts) return ERR_INVALID;
    const route_plan p = {nullptr, (unsigned)num_experts, (unsigned)choices, 1, 1, 1, scores == TB200_SIGMOID, renormalize != 0, scale};
    const bool dense = scores == TB200_SOFTMAX && !renormalize;
    auto go = [&](auto vv, auto lanes) -> int {
      constexpr int V = decltype(vv)::value, L = decltype(lanes)::value, TOKENS = BLOCK / L;
      (dense ? expert_route_grad_kernel<T, L, V, true> : expert_route_grad_kernel<T, L, V, false>)<<<(unsigned)((n + TOKENS - 1) / TOKENS), BLOCK, 0, stream>>>(
          d_dweights, d_experts, static_cast<const T*>(d_logits), logits_stride, (unsigned)n, p, static_cast<T*>(d_dlogits));
      return (int)cudaGetLastError();
    };
    auto with = [&](auto vv) -> int { return choices <= 8 && num_experts <= 64 ? go(vv, std::integral_constant<int, 8>()) : go(vv, std::integral_constant<int, 32>()); };
    if ((!dense || in_16_bytes(d_logits, num_experts, logits_stride, sizeof(T))) && in_16_bytes(d_dlogits, num_experts, num_experts, sizeof(T)))
      return with(std::integral_constant<int, 16 / sizeof(T)>());
    return with(std::integral_constant<int, 1>());
  });
}
