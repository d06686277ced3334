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

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
template <class R> __device__ __forceinline__ R lowest() { return -(R)INFINITY; }

// the largest of the warp's values; an order on floats that the warp's integer reduction knows (no NaNs come here, no -0 either)
__device__ __forceinline__ unsigned ordered(float x) { const unsigned u = __float_as_uint(x); return u & 0x80000000u ? ~u : u | 0x80000000u; }
__device__ __forceinline__ float warp_max(float x) {
  const unsigned u = __reduce_max_sync(ALL, ordered(x));
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
template <class R> __device__ __forceinline__ R warp_sum(R x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
  return x;
}
__device__ __forceinline__ double warp_max(double x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) { const double y = __shfl_xor_sync(ALL, x, o); x = y > x ? y : x; }
  return x;
}

// Of the softmax over a row's open experts: its largest logit and the sum of exp(logit - largest).  An infinite logit leaves the others nothing.
template <class R> struct softmax_of {
  R top, sum;
  __device__ __forceinline__ R share(R x) const { return x == top ? (R)1 : exp_of(x - top); }      // times the sum
};
template <class R> __device__ __forceinline__ R sigmoid_of(R x) { return (R)1 / ((R)1 + exp_of(-x)); }

template <class R> struct best_of { R value; int at; };
// The best of a row's experts in [low, high) other than `but`, the first of equal ones; value -inf and no place where there is none.
template <class R, int PER> __device__ __forceinline__ best_of<R> warp_best(const R (&order)[PER], int low, int high, int but) {
  const int lane = threadIdx.x % 32;
  R mine = lowest<R>();
  int at = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    if (order[i] > mine && e >= low && e < high && e != but) { mine = order[i]; at = e; }
  }
  best_of<R> b;
  b.value = warp_max(mine);
  b.at = (int)__reduce_min_sync(ALL, mine == b.value ? (unsigned)at : 0x7fffffffu);
  return b;
}

// The choices of one row, choice c in lane c (-1: none), found by a warp that holds expert i * 32 + lane in order[i].
//
// Scores are compared as 64-bit numbers would be.  Where the order is the logits' (no bias, and no sums of scores of groups) it is exact as it is.
// Otherwise the scores are 32-bit numbers that are off by up to `slack`: two neighbours in the order that are nearer than that, and the last group
// kept and the first left out, are `unsure`, and the row is done again in 64 bits.  (Equal logits with equal biases are as equal there.)  Every
// row in 64 bits takes three times as long.
template <class R, int PER, class T> __device__ __forceinline__ bool choose(const route_plan& p, const T* row, int& chosen, softmax_of<R>& all) {
  const int lane = threadIdx.x % 32;
  const int experts = (int)p.experts;
  const bool sums = p.groups > 1 && p.group_best > 1, exact = sizeof(R) == 8 || (!p.bias && !sums);
  R order[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    const float x = e < experts ? to_f32(row[e]) : -INFINITY;
    order[i] = x > -INFINITY ? (R)x + (R)0 : lowest<R>();      // neither NaN nor -0
  }
  all.top = lowest<R>();
  all.sum = (R)1;
  if (!p.sigmoid && (!p.renormalize || p.bias || sums)) {
    R mine = lowest<R>(), sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine = order[i] > mine ? order[i] : mine;
    all.top = warp_max(mine);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (order[i] > lowest<R>()) sum += all.share(order[i]);
    all.sum = warp_sum(sum);
  }
  auto score = [&](R x) { return p.sigmoid ? sigmoid_of(x) : all.share(x) / all.sum; };
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (order[i] > lowest<R>()) {
        const R v = score(order[i]) + (R)p.bias[i * 32 + lane];
        order[i] = v > lowest<R>() ? v + (R)0 : lowest<R>();
      }
  }
  // sums of up to 1024 exponentials, whose arguments are rounded differences: good to 2^-18 of the largest score; a sum with a bias to 2^-24 of itself
  const R largest = p.sigmoid ? (R)1 : (R)1 / all.sum;
  auto slack = [&](R v) { return (R)0x1p-18 * largest + (R)0x1p-22 * (v < 0 ? -v : v); };
  bool unsure = false;
  if (p.groups > 1) {
    const int size = experts / (int)p.groups;
    R mine = lowest<R>();
    for (int g = 0; g < (int)p.groups; ++g) {
      const best_of<R> first = warp_best<R, PER>(order, g * size, (g + 1) * size, -1);
      R sum = first.value;
      if (sums && first.value > lowest<R>()) {
        const best_of<R> second = warp_best<R, PER>(order, g * size, (g + 1) * size, first.at);
        sum = p.bias ? first.value : score(first.value);
        if (second.value > lowest<R>()) sum += p.bias ? second.value : score(second.value);
        sum += (R)0;
      }
      if (lane == g) mine = sum;
    }
    int before = 0;
    for (int g = 0; g < (int)p.groups; ++g) {
      const R other = __shfl_sync(ALL, mine, g);
      before += other > mine || (other == mine && g < lane);
    }
    const bool stays = lane < (int)p.groups && before < (int)p.group_choices;
    const unsigned kept = __ballot_sync(ALL, stays);
    if (!exact) {
      const R last = -warp_max(stays ? -mine + (R)0 : lowest<R>()), next = warp_max(stays ? lowest<R>() : mine);
      if (next > lowest<R>() && last - next < 2 * slack(last)) unsure = true;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * 32 + lane;
      if (e < experts && !(kept >> (e / size) & 1)) order[i] = lowest<R>();
    }
  }
  chosen = -1;
  best_of<R> last = {(R)0, -1};
  for (int c = 0; c < (int)p.choices + (exact ? 0 : 1); ++c) {
    const best_of<R> next = warp_best<R, PER>(order, 0, experts, -1);
    if (!(next.value > lowest<R>())) break;
    if (!exact && c > 0 && last.value - next.value < slack(last.value)) {
      const float x = to_f32(row[last.at]), y = to_f32(row[next.at]);
      unsure |= !(x == y && (!p.bias || p.bias[last.at] == p.bias[next.at]));
    }
    if (lane == c && c < (int)p.choices) chosen = next.at;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * 32 + lane == next.at) order[i] = lowest<R>();
    last = next;
  }
  return unsure;
}
// (not inlined: few rows come here, and its registers would be all rows')
template <int PER, class T> __device__ __noinline__ int choose_in_64(const route_plan& p, const T* row) {
  int chosen;
  softmax_of<double> all;
  choose<double, PER>(p, row, chosen, all);
  return chosen;
}

// w = scale * score (/ the sum of the chosen ones' scores) of the chosen expert's logit x.  Quotients are made of exponentials relative to the largest, so that
// they hold where the scores themselves vanish: with c = min(largest, 0), sigmoid(x) e^-c = e^(x - c) / (1 + e^x) for x <= 0.
struct weight_of { float w, other; };      // the quotient or the score; 1 - sigmoid(x)
__device__ __forceinline__ weight_of weigh(bool chosen, float x, bool sigmoid, bool renormalize, const softmax_of<float>& all) {
  weight_of r = {0.f, 0.f};
  if (sigmoid) {
    const float e = expf(-fabsf(x));
    r.other = x >= 0.f ? e / (1.f + e) : 1.f / (1.f + e);
    if (!renormalize) {
      r.w = x >= 0.f ? 1.f / (1.f + e) : e / (1.f + e);
    } else {
      const float c = fminf(warp_max(chosen ? x + 0.f : -INFINITY), 0.f);
      r.w = x > 0.f ? 1.f / (1.f + e) : (x == c ? 1.f : expf(x - c)) / (1.f + e);
    }
  } else if (renormalize) {
    softmax_of<float> some = {warp_max(chosen ? x + 0.f : -INFINITY), 1.f};
    r.w = some.share(x);
  } else {
    r.w = all.share(x) / all.sum;
  }
  if (!chosen) r.w = 0.f;
  if (renormalize) {
    const float sum = warp_sum(r.w);
    r.w = sum > 0.f ? r.w / sum : 0.f;
  }
  return r;
}

// A warp a token.  Bound by how long its choices take one after another (each a comparison of what the lanes hold and two reductions).
template <class T, int PER>
__global__ void __launch_bounds__(BLOCK) expert_route_kernel(const T* __restrict__ logits, size_t stride, unsigned n, route_plan p, int* __restrict__ experts, float* __restrict__ weights) {
  const unsigned token = blockIdx.x * (BLOCK / 32) + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (token >= n) return;
  const T* const row = logits + token * stride;
  int chosen;
  softmax_of<float> all;
  if (choose<float, PER>(p, row, chosen, all)) chosen = choose_in_64<PER>(p, row);
  const float x = chosen >= 0 ? to_f32(row[chosen]) : 0.f;
  const weight_of r = weigh(chosen >= 0, x, p.sigmoid, p.renormalize, all);
  if (lane < p.choices) {
    experts[(size_t)token * p.choices + lane] = chosen;
    weights[(size_t)token * p.choices + lane] = p.scale * r.w;
  }
}

// A warp a token: what every expert's logit gets (zero but for the whole softmax), then the chosen ones' in their places.
//   renormalised: w_c (g_c - sum of g w) (sigmoid: times 1 - s_c);   softmax: p_e (G_e - sum of g p);   sigmoid: g_c s_c (1 - s_c),
// with G_e the sum of g over the choices of e.  Bound by the launch and, from some thousand tokens on, by the bytes of dlogits.
template <class T, int V, bool DENSE>
__global__ void __launch_bounds__(BLOCK) expert_route_grad_kernel(const float* __restrict__ dweights, const int* __restrict__ ids, const T* __restrict__ logits, size_t stride, unsigned n,
                                                                route_plan p, T* __restrict__ dlogits) {
  const unsigned token = blockIdx.x * (BLOCK / 32) + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (token >= n) return;
  const T* const row = logits + token * stride;
  T* const to = dlogits + (size_t)token * p.experts;
  const unsigned pieces = p.experts / V;
  const int id = lane < p.choices ? ids[(size_t)token * p.choices + lane] : -1;
  float x = (unsigned)id < p.experts ? to_f32(row[id]) : -INFINITY;
  const bool chosen = x > -INFINITY;
  x = chosen ? x : 0.f;
  const float g = chosen ? p.scale * dweights[(size_t)token * p.choices + lane] : 0.f;
  softmax_of<float> all = {-INFINITY, 1.f};
  if (DENSE) {
    float top = -INFINITY, sum = 0.f;
    for (unsigned c = lane; c < pieces; c += 32) {
      float f[V];
      channels(load_words<T, V>(row + c * V), f);
#pragma unroll
      for (int v = 0; v < V; ++v) top = f[v] > top ? f[v] : top;
    }
    all.top = warp_max(top + 0.f);
    for (unsigned c = lane; c < pieces; c += 32) {
      float f[V];
      channels(load_words<T, V>(row + c * V), f);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (f[v] > -INFINITY) sum += all.share(f[v]);
    }
    all.sum = warp_sum(sum);
  }
  const weight_of r = weigh(chosen, x, p.sigmoid, p.renormalize, all);
  const float mean = p.renormalize || DENSE ? warp_sum(g * r.w) : 0.f;
  // of this choice; choices of the same expert are added up, in their order
  const float own = DENSE ? g : p.renormalize ? r.w * (g - mean) * (p.sigmoid ? r.other : 1.f) : g * r.w * r.other;
  float d = 0.f;
  for (unsigned c = 0; c < p.choices; ++c) {
    const int other = __shfl_sync(ALL, chosen ? id : -1, c);
    const float add = __shfl_sync(ALL, own, c);
    if (other == id) d += add;
  }
  if (DENSE) d = r.w * (d - mean);
  for (unsigned c = lane; c < pieces; c += 32) {
    float f[V];
    if (DENSE) channels(load_words<T, V>(row + c * V), f);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = DENSE && f[v] > -INFINITY ? -(all.share(f[v]) / all.sum) * mean : 0.f;
    store_words<T, V>(to + c * V, to_words<T, V>(f));
  }
  __syncwarp();
  if (chosen) to[id] = from_f32<T>(d);
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
    auto go = [&](auto per) -> int {
      expert_route_kernel<T, decltype(per)::value><<<(unsigned)((n + BLOCK / 32 - 1) / (BLOCK / 32)), BLOCK, 0, stream>>>(static_cast<const T*>(d_logits), logits_stride, (unsigned)n, p, d_experts,
                                                                                                                 d_weights);
      return (int)cudaGetLastError();
    };
    if (num_experts <= 32) return go(std::integral_constant<int, 1>());
    if (num_experts <= 64) return go(std::integral_constant<int, 2>());
    if (num_experts <= 128) return go(std::integral_constant<int, 4>());
    if (num_experts <= 256) return go(std::integral_constant<int, 8>());
    if (num_experts <= 512) return go(std::integral_constant<int, 16>());
    return go(std::integral_constant<int, 32>());
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
    auto go = [&](auto vv) -> int {
      constexpr int V = decltype(vv)::value;
      (dense ? expert_route_grad_kernel<T, V, true> : expert_route_grad_kernel<T, V, false>)<<<(unsigned)((n + BLOCK / 32 - 1) / (BLOCK / 32)), BLOCK, 0, stream>>>(
          d_dweights, d_experts, static_cast<const T*>(d_logits), logits_stride, (unsigned)n, p, static_cast<T*>(d_dlogits));
      return (int)cudaGetLastError();
    };
    if ((!dense || in_16_bytes(d_logits, num_experts, logits_stride, sizeof(T))) && in_16_bytes(d_dlogits, num_experts, num_experts, sizeof(T)))
      return go(std::integral_constant<int, 16 / sizeof(T)>());
    return go(std::integral_constant<int, 1>());
  });
}
