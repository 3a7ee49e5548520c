// Routing of tokens to experts and its gradient: one warp per token, the token's logits in registers (a lane holds VPL
// neighbouring experts).  Forward and backward read every logit once; bytes bound long batches, launch latency short
// ones.
//
// The choice is defined on exact scores, so that neither the type nor the rounding of a softmax decides between two
// experts.  Without bias and groups both scorings are monotone and the logits themselves are compared.  Otherwise
// scores are computed in fp32 with a bound on their error; where two values that decide the result lie closer than
// that bound, the warp computes the row's scores again in 64 bits and chooses by those.
//
// A lane's values become whole numbers in their order whose lowest bits are the value's place in the lane, and a
// sorting network puts them in descending order once; every one of the top_k rounds then is a maximum over 32 heads and
// a shift in the winning lane.  The bits given to the place widen the distance that counts as near.
//
// Measured (fp32 logits, device time): 16384 x 256 in 8 groups of which 4 stay, sigmoid with bias, top 8: 23.8 us, where
// reading the rows takes 2.7: bound by the latency of the choice (a reduction, a vote and a shift per round) at 40 warps an
// SM; without bias and groups 14.4 us; 16384 x 64 softmax, top 6: 11.7 us; 16 x 64: 2.9 us, one launch.
// A row that needs 64 bits adds 4.6 us of latency to the launch that meets it.  3 in 1000 rows of the first case do, so it is
// the launch's tail, not its sum.  More do where scores come from 16-bit logits that tie, in groups and without a bias: 32 %
// of normal bf16 rows of that size (fp16 5 %), 42.6 us (26.8) instead of 22.2; 13 % of 64 experts, 17.5 instead of 13.7.  All
// do where a large finite bias masks experts, since the bound grows with it (-1e4 or -1e9: 64 us, 27 for 64 experts; a mask
// of -inf costs nothing), and where neither a score nor the bias reaches 2e-3 (the same times).
#include "ftb_lm.cuh"

namespace ftb {

constexpr int kMaxGroups = 32;  // a lane holds a group's value
constexpr unsigned kAll = 0xffffffffu;

struct RouteArgs {
  const void* logits;
  const float* bias;
  int* ids;
  float* weights;
  const float* dweights;
  void* dlogits;
  long long tokens;
  int experts, top_k, scoring, groups, top_groups, renorm, vec;
  int group_lanes;  // lanes of a group where every lane's experts share one and the lanes are a power of two, else 0
  float scale;
};

template <typename T>
__device__ __forceinline__ float load_logit(const T* p);
template <>
__device__ __forceinline__ float load_logit<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float load_logit<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <>
__device__ __forceinline__ float load_logit<__half>(const __half* p) { return __half2float(*p); }

__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_logit(__half* p, float v) { *p = __float2half_rn(v); }

// NaN counts as -inf (the larger of it and -inf is the latter); -0 becomes 0, which orders equal to it.
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY) + 0.0f; }

// The lane's VPL logits; -inf past the last expert.
template <typename T, int VPL>
__device__ __forceinline__ void load_row(const T* row, int experts, int lane, bool vec, float (&x)[VPL]) {
  const int e0 = lane * VPL;
  constexpr int PER = 16 / static_cast<int>(sizeof(T));
  if constexpr (VPL % PER == 0) {
    if (vec && e0 + VPL <= experts) {
#pragma unroll
      for (int q = 0; q < VPL / PER; ++q) {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + e0 + q * PER);
        const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < PER; ++i) x[q * PER + i] = clean(load_logit<T>(t + i));
      }
      return;
    }
  }
#pragma unroll
  for (int v = 0; v < VPL; ++v) x[v] = e0 + v < experts ? clean(load_logit<T>(row + e0 + v)) : -INFINITY;
}

template <typename S>
__device__ __forceinline__ S warp_sum(S v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}

// Whole numbers in the order of the floating values (never 0, which stands for "none left").
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t order_key(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v));
  return b ^ ((b >> 63) ? ~0ull : (1ull << 63));
}
__device__ __forceinline__ double key_value(uint64_t k) {
  return __longlong_as_double(static_cast<long long>(k ^ ((k >> 63) ? (1ull << 63) : ~0ull)));
}
__device__ __forceinline__ uint32_t key_max(uint32_t k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ uint64_t key_max(uint64_t k) {
  const uint32_t hi = __reduce_max_sync(kAll, static_cast<uint32_t>(k >> 32));
  const uint32_t lo = __reduce_max_sync(kAll, (k >> 32) == hi ? static_cast<uint32_t>(k) : 0u);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

__device__ __forceinline__ float warp_max(float v) { return key_value(key_max(order_key(v))); }

// The `count` largest of a lane's keys (0: not there), best first, ties to the lowest index: lane j gets the index of
// the j-th.
template <typename K, int VPL>
__device__ __forceinline__ int pick(K (&k)[VPL], int count, int lane) {
  int mine = 0;
  for (int j = 0; j < count; ++j) {
    K best = k[0];
    int at = 0;
#pragma unroll
    for (int v = 1; v < VPL; ++v)
      if (k[v] > best) {
        best = k[v];
        at = v;
      }
    const K top = key_max(best);
    const int winner = __ffs(__ballot_sync(kAll, best == top)) - 1;
    const int id = __shfl_sync(kAll, lane * VPL + at, winner);
    if (lane == j) mine = id;
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if (lane == winner && v == at) k[v] = 0;
  }
  return mine;
}

template <typename S>
__device__ __forceinline__ void merge_top2(S& a, S& b, S oa, S ob) {
  // the two largest of two ordered pairs
  const S lo = a > oa ? oa : a;
  a = a > oa ? a : oa;
  b = b > ob ? b : ob;
  b = b > lo ? b : lo;
}

// The best top_groups of the values that the lanes hold (`there`: the lane holds one), as a mask of lanes; ties to the
// lowest lane.  `near` is set where the last kept and the first left out are within `tol`.
template <typename S>
__device__ __forceinline__ uint32_t best_lanes(S value, bool there, int count, S tol, int lane, bool* near) {
  if (value != value) value = static_cast<S>(-INFINITY);
  auto key = order_key(value);
  if (!there) key = 0;
  auto last = key;
  uint32_t kept = 0;
  for (int j = 0; j < count; ++j) {
    last = key_max(key);
    const uint32_t tied = __ballot_sync(kAll, key == last), lowest = tied & (0u - tied);
    kept |= lowest;
    if ((lowest >> lane) & 1u) key = 0;
  }
  const auto rest = key_max(key);
  if (rest != 0) *near |= key_value(last) - key_value(rest) <= tol;
  return kept;
}

// Bits of the lane's values that lie in the kept groups.
template <typename S, int VPL>
__device__ __forceinline__ uint32_t keep_groups(const RouteArgs& p, const S (&c)[VPL], uint32_t avail, S tol, int lane,
                                                bool* near) {
  const S none = static_cast<S>(-INFINITY);
  if (p.group_lanes > 0) {
    // a group is a run of lanes
    S a = none, b = none;
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if ((avail >> v) & 1u) merge_top2(a, b, c[v], none);
    for (int d = 1; d < p.group_lanes; d <<= 1) merge_top2(a, b, __shfl_xor_sync(kAll, a, d), __shfl_xor_sync(kAll, b, d));
    const int first = lane & ~(p.group_lanes - 1);
    const uint32_t kept = best_lanes<S>(p.group_lanes * VPL > 1 ? a + b : a, lane == first && lane * VPL < p.experts, p.top_groups, tol, lane, near);
    return (kept >> first) & 1u ? avail : 0u;
  }
  const int size = p.experts / p.groups, e0 = lane * VPL;
  S value = none;  // of group `lane`
  for (int g = 0; g < p.groups; ++g) {
    S a = none, b = none;
#pragma unroll
    for (int v = 0; v < VPL; ++v)
      if (((avail >> v) & 1u) && e0 + v >= g * size && e0 + v < (g + 1) * size) merge_top2(a, b, c[v], none);
#pragma unroll
    for (int d = 16; d; d >>= 1) merge_top2(a, b, __shfl_xor_sync(kAll, a, d), __shfl_xor_sync(kAll, b, d));
    if (lane == g) value = size > 1 ? a + b : a;
  }
  const uint32_t kept = best_lanes<S>(value, lane < p.groups, p.top_groups, tol, lane, near);
  uint32_t left = 0;
  int g = e0 / size, end = (g + 1) * size;
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    if (e0 + v >= end) {
      ++g;
      end += size;
    }
    if (((avail >> v) & 1u) && ((kept >> g) & 1u)) left |= 1u << v;
  }
  return left;
}

// exp(x - m) with the limits that a row of infinities has: the largest share the mass, a row of -inf has none.
__device__ __forceinline__ float exp_below(float x, float m) { return m == -INFINITY ? 0.0f : x == m ? 1.0f : expf(x - m); }

template <int VPL>
__device__ __noinline__ int choose_exactly(const RouteArgs& p, const float (&x)[VPL], uint32_t avail, float m, int lane) {
  if (!p.bias && p.groups == 1) {
    uint32_t k[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) k[v] = (avail >> v) & 1u ? order_key(x[v]) : 0u;
    return pick<uint32_t, VPL>(k, p.top_k, lane);
  }
  double c[VPL];
  double sum = 0.0;
  const int e0 = lane * VPL;
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    const double d = static_cast<double>(x[v]);
    if (p.scoring == FTB_SCORE_SIGMOID) c[v] = 1.0 / (1.0 + exp(-d));
    else c[v] = m == -INFINITY ? 0.0 : x[v] == m ? 1.0 : exp(d - static_cast<double>(m));
    sum += ((avail >> v) & 1u) ? c[v] : 0.0;
  }
  sum = warp_sum(sum);
#pragma unroll
  for (int v = 0; v < VPL; ++v) {
    if (p.scoring == FTB_SCORE_SOFTMAX) c[v] = sum > 0.0 ? c[v] / sum : 0.0;
    if (p.bias && ((avail >> v) & 1u)) c[v] += static_cast<double>(p.bias[e0 + v]);
    c[v] = c[v] != c[v] ? -INFINITY : c[v] + 0.0;
  }
  bool near = false;
  if (p.groups > 1) avail = keep_groups<double, VPL>(p, c, avail, -1.0, lane, &near);
  uint64_t k[VPL];
#pragma unroll
  for (int v = 0; v < VPL; ++v) k[v] = (avail >> v) & 1u ? order_key(c[v]) : 0ull;
  return pick<uint64_t, VPL>(k, p.top_k, lane);
}

// Batcher's odd-even merge sort of N keys in registers, largest first.
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int d = p; d > 0; d /= 2)
#pragma unroll
      for (int j = d % p; j + d < N; j += 2 * d)
#pragma unroll
        for (int i = 0; i < d; ++i)
          if (i + j + d < N && (i + j) / (2 * p) == (i + j + d) / (2 * p)) {
            const uint32_t a = k[i + j], b = k[i + j + d];
            k[i + j] = max(a, b);
            k[i + j + d] = min(a, b);
          }
}

// pick() on sorted keys; `gap` becomes the least distance between neighbours in the order of choice, the last chosen and
// the first left out among them (0 for values that differ in the place's bits only).  TIES: equal values go to the lowest
// index, which the place's bits alone do not say across lanes; without it the caller looks again where the gap is 0.
template <int VPL, bool TIES>
__device__ __forceinline__ int pick_sorted(uint32_t (&k)[VPL], int count, int lane, float* gap) {
  constexpr uint32_t PLACE = VPL - 1;
  int mine = 0;
  uint32_t taken = 0;  // lane j: the j-th key
  for (int j = 0; j < count; ++j) {
    const uint32_t head = TIES ? k[0] & ~PLACE : k[0], top = __reduce_max_sync(kAll, head);
    const int winner = __ffs(__ballot_sync(kAll, head == top)) - 1;
    const uint32_t full = TIES ? __shfl_sync(kAll, k[0], winner) : top;
    if (lane == j) {
      taken = top;
      mine = winner * VPL + static_cast<int>(PLACE - (full & PLACE));
    }
    const bool pop = lane == winner;
#pragma unroll
    for (int v = 0; v + 1 < VPL; ++v) k[v] = pop ? k[v + 1] : k[v];
    k[VPL - 1] = pop ? 0u : k[VPL - 1];
  }
  // lane j: the j-th key and the one before it; lane `count` (or, past lane 31, every lane) the first left out
  const uint32_t rest = __reduce_max_sync(kAll, k[0]) & ~PLACE;
  taken &= ~PLACE;
  const uint32_t last = __shfl_sync(kAll, taken, count - 1);
  uint32_t before = __shfl_up_sync(kAll, taken, 1), key = taken;
  if (lane == 0 || lane >= count) {
    before = last;
    key = rest;
  }
  // equal infinities are 0 apart; the difference of an infinity and anything else says nothing and is far enough
  float apart = key == before ? 0.0f : key_value(before) - key_value(key);
  if (key == 0 || apart != apart) apart = INFINITY;
  *gap = __uint_as_float(__reduce_min_sync(kAll, __float_as_uint(apart)));
  return mine;
}

// The groups kept, where a group is a run of p.group_lanes lanes: from the two largest keys of every lane.  Returns
// whether the lane's group stays; `near` where the last group kept and the first left out are within `tol`.
template <int VPL>
__device__ __forceinline__ bool keep_lane_groups(const RouteArgs& p, const uint32_t (&k)[VPL], float tol, int lane, bool* near) {
  constexpr uint32_t PLACE = VPL - 1;
  // (the key of -inf without its place's bits is none: clean)
  float a = clean(key_value(k[0] & ~PLACE)), b = VPL > 1 ? clean(key_value(k[VPL > 1 ? 1 : 0] & ~PLACE)) : -INFINITY;
  for (int d = 1; d < p.group_lanes; d <<= 1) merge_top2(a, b, __shfl_xor_sync(kAll, a, d), __shfl_xor_sync(kAll, b, d));
  const int first = lane & ~(p.group_lanes - 1);
  const uint32_t kept = best_lanes<float>(p.group_lanes * VPL > 1 ? a + b : a, lane == first && lane * VPL < p.experts, p.top_groups, tol, lane, near);
  return (kept >> first) & 1u;
}

// FULL: every lane has VPL experts, and the rows and the bias can be read in 16-byte words.
// The loop over the choices waits for its reductions, so warps count: registers are held to what lets 8 blocks run on
// an SM (5 with 8 experts per lane): 16384 x 64, top 6: 15.4 -> 13.4 us; 16384 x 256 in groups, top 8: 26.5 -> 24.5.
template <typename T, int VPL, bool FULL>
__global__ void __launch_bounds__(256, VPL <= 4 ? 8 : VPL == 8 ? 5 : 1) route_kernel(const RouteArgs p) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long t = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (t >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.experts;
  const int e0 = lane * VPL;
  float x[VPL];
  load_row<T, VPL>(row, p.experts, lane, FULL || p.vec != 0, x);
  const int have = FULL ? VPL : min(max(p.experts - e0, 0), VPL);
  const uint32_t avail = have >= 32 ? kAll : (1u << have) - 1u;

  const bool sigmoid = p.scoring == FTB_SCORE_SIGMOID;
  const bool by_logit = !p.bias && p.groups == 1;
  float m = -INFINITY, total = 0.0f;
  if (!sigmoid) {
#pragma unroll
    for (int v = 0; v < VPL; ++v) m = fmaxf(m, x[v]);
    m = warp_max(m);
  }
  constexpr uint32_t PLACE = VPL - 1;
  uint32_t k[VPL];
  int mine;
  bool near = false;
  if (by_logit) {
#pragma unroll
    for (int v = 0; v < VPL; ++v) k[v] = FULL || v < have ? (order_key(x[v]) & ~PLACE) | (PLACE - v) : 0u;
    sort_keys<VPL>(k);
    float gap;
    mine = pick_sorted<VPL, sizeof(T) == 2>(k, p.top_k, lane, &gap);
    // A 16-bit logit has no bits where the place goes, so equal keys are equal logits.  An fp32 one may differ in the
    // bits that the place took: look again where two keys agree but for them.
    if (sizeof(T) == 4) near = !(gap > 0.0f);
    if (!sigmoid && !p.renorm) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) total += exp_below(x[v], m);
      total = warp_sum(total);
    }
  } else {
    float c[VPL];
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      c[v] = sigmoid ? __fdividef(1.0f, 1.0f + __expf(-x[v])) : exp_below(x[v], m);
      if (!FULL && v >= have) c[v] = 0.0f;
    }
    if (!sigmoid) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) total += c[v];
      total = warp_sum(total);
      const float inv = total > 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
      for (int v = 0; v < VPL; ++v) c[v] *= inv;
    }
    float most = 0.0f;  // largest magnitude that enters a sum: what the error bound scales with
#pragma unroll
    for (int v = 0; v < VPL; ++v) most = fmaxf(most, c[v]);
    if (p.bias) {
      float b[VPL];
      load_row<float, VPL>(p.bias, p.experts, lane, FULL, b);
#pragma unroll
      for (int v = 0; v < VPL; ++v) {
        const float size = fabsf(b[v]);
        most = fmaxf(most, size < INFINITY ? size : 0.0f);
        c[v] = clean(c[v] + b[v]);
      }
    }
    // What two compared values may be off by, relative to `most`.  softmax: the largest score is at least 1 / experts of
    // the sum, its exponential and those below it are good to 2 units of 2^-23 of themselves, the sum over the row to
    // about 8.  sigmoid: the fast exponential is good to 2 + 1.173 |x| units of 2^-23, the reciprocal to 2, so a score is
    // off by at most 1.4e-6 of the largest one while that is at least sigmoid(-6.2) = 2e-3 (scores below it are off by
    // more of themselves, but they are smaller by more than that); two of them by 2.8e-6, two sums of two by 5.6e-6, and
    // adding the bias and the two rounds each value by 2^-24 of up to 4 `most`.  Where every score is smaller and no bias
    // is larger, the bound is lost (at -87.3 the reciprocal is 0) and 64 bits decide.  The place takes VPL units of a value
    // of up to twice `most`.
    most = __uint_as_float(__reduce_max_sync(kAll, __float_as_uint(most)));
    const float tol = (3.2e-6f + VPL * 2.4e-7f) * most;
    near = sigmoid && most < 2e-3f;
    uint32_t left = avail;
    if (p.groups > 1 && p.group_lanes == 0) left = keep_groups<float, VPL>(p, c, avail, 2.0f * tol, lane, &near);
#pragma unroll
    for (int v = 0; v < VPL; ++v) k[v] = (order_key(c[v]) & ~PLACE) | (PLACE - v);
    if (left != (VPL == 32 ? kAll : (1u << (VPL & 31)) - 1u)) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) k[v] = (left >> v) & 1u ? k[v] : 0u;
    }
    sort_keys<VPL>(k);
    if (p.groups > 1 && p.group_lanes > 0 && !keep_lane_groups<VPL>(p, k, 2.0f * tol, lane, &near)) {
#pragma unroll
      for (int v = 0; v < VPL; ++v) k[v] = 0;
    }
    float gap;
    mine = pick_sorted<VPL, false>(k, p.top_k, lane, &gap);
    near |= !(gap > tol);
  }
  if (near) mine = choose_exactly<VPL>(p, x, avail, m, lane);

  // weights: lane j < top_k has the j-th expert
  const bool active = lane < p.top_k;
  const float l = active ? clean(load_logit<T>(row + mine)) : -INFINITY;
  float w;
  if (sigmoid) {
    w = active ? 1.0f / (1.0f + expf(-l)) : 0.0f;
    if (p.renorm) {
      float s = warp_sum(w);
      if (s < 1e-30f) {
        // every chosen score underflows or nearly so: the ratios of exp(l), which 1 / (1 + exp(-l)) tends to
        const float top = warp_max(l);
        w = active ? exp_below(l, top) : 0.0f;
        s = warp_sum(w);
      }
      w = s > 0.0f ? w / s : 0.0f;
    }
  } else if (p.renorm) {
    const float top = warp_max(l);
    w = active ? exp_below(l, top) : 0.0f;
    const float s = warp_sum(w);
    w = s > 0.0f ? w / s : 0.0f;
  } else {
    w = total > 0.0f ? exp_below(l, m) / total : 0.0f;
  }
  if (active) {
    p.ids[t * p.top_k + lane] = mine;
    p.weights[t * p.top_k + lane] = w * p.scale;
  }
}

// d logits.  With the chosen scores scaled to one, r = s / S with S the sum of the chosen s, softmax gives
//   dl_j = r_j g_j with g_j = scale (dw_j - sum_i r_i dw_i)
// for the chosen (the row's other logits cancel), and sigmoid dl_j = r_j g_j (1 - s_j), taken as (dw_j - sum dw s / S) / S s_j
// while S is 1e-9 or more and by the ratios of exp(l) below that.  Without scaling softmax gives dl_e = s_e (g_e -
// sum_j g_j s_j) for every expert and sigmoid dl_j = g_j s_j (1 - s_j), g = scale dw.  An expert that a row names twice gets
// both parts, added in the order of the slots.  8192 x 128 bf16, softmax over all: 5 us of device time for 4.7 MB.
template <typename T, int VPL>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteArgs p) {
  grid_dependency_wait();
  grid_launch_dependents();
  __shared__ float grad[8][32 * VPL];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long t = static_cast<long long>(blockIdx.x) * 8 + warp;
  if (t >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + t * p.experts;
  T* drow = static_cast<T*>(p.dlogits) + t * p.experts;
  const int e0 = lane * VPL;
  const bool sigmoid = p.scoring == FTB_SCORE_SIGMOID;
  int id = lane < p.top_k ? p.ids[t * p.top_k + lane] : -1;
  const bool active = id >= 0 && id < p.experts;
  if (!active) id = 0;
  const float dw = active ? p.dweights[t * p.top_k + lane] * p.scale : 0.0f;
  const float l = active ? clean(load_logit<T>(row + id)) : -INFINITY;
  const bool full = !sigmoid && !p.renorm;  // every logit has a gradient
  float x[VPL];
  float m = -INFINITY, total = 0.0f;
  if (full) {
    load_row<T, VPL>(row, p.experts, lane, p.vec != 0, x);
#pragma unroll
    for (int v = 0; v < VPL; ++v) m = fmaxf(m, x[v]);
    m = warp_max(m);
#pragma unroll
    for (int v = 0; v < VPL; ++v) {
      x[v] = exp_below(x[v], m);
      total += x[v];
    }
    total = warp_sum(total);
  }
  float part;  // what the lane's slot adds to its expert's gradient (full: its g)
  float back = 0.0f;
  if (full) {
    const float inv = total > 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
    for (int v = 0; v < VPL; ++v) x[v] *= inv;
    part = dw;
    back = warp_sum(active ? dw * exp_below(l, m) * inv : 0.0f);
  } else {
    const float s = sigmoid ? (active ? 1.0f / (1.0f + expf(-l)) : 0.0f) : 0.0f;
    if (p.renorm) {
      const float sum = sigmoid ? warp_sum(s) : 0.0f;
      if (sum >= 1e-9f) {
        part = (dw - warp_sum(dw * s) / sum) / sum * s;
      } else {
        // softmax, or scores below 1e-9, which are exp(l) to 1e-9 of themselves: by the ratios of exp(l), so that neither
        // dw s leaves the range of fp32 nor dw / sum
        const float top = warp_max(l);
        float r = active ? exp_below(l, top) : 0.0f;
        const float total_r = warp_sum(r);
        r = total_r > 0.0f ? r / total_r : 0.0f;
        const float mean = warp_sum(r * dw);
        part = active ? r * (dw - mean) : 0.0f;
      }
    } else {
      part = s * dw;
    }
    // 1 - s without cancellation
    if (sigmoid) part = active ? part * (1.0f / (1.0f + expf(l))) : 0.0f;
  }
  float* mine = grad[warp];
#pragma unroll
  for (int v = 0; v < VPL; ++v) mine[v * 32 + lane] = 0.0f;
  __syncwarp();
  for (int j = 0; j < p.top_k; ++j) {
    if (lane == j && active) mine[id] += part;
    __syncwarp();
  }
#pragma unroll
  for (int v = 0; v < VPL; ++v) x[v] = full ? x[v] * (mine[e0 + v] - back) : mine[e0 + v];
  constexpr int PER = 16 / static_cast<int>(sizeof(T));
  if constexpr (VPL % PER == 0) {
    if (p.vec && e0 + VPL <= p.experts) {
#pragma unroll
      for (int q = 0; q < VPL / PER; ++q) {
        uint4 raw;
        T* o = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int i = 0; i < PER; ++i) store_logit(o + i, x[q * PER + i]);
        *reinterpret_cast<uint4*>(drow + e0 + q * PER) = raw;
      }
      return;
    }
  }
#pragma unroll
  for (int v = 0; v < VPL; ++v)
    if (e0 + v < p.experts) store_logit(drow + e0 + v, x[v]);
}

template <typename T, int VPL>
static int launch_route(const RouteArgs& p, bool backward, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.tokens + 7) / 8));
  const bool full = p.experts == 32 * VPL && p.vec && (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0;
  auto kern = backward ? route_backward_kernel<T, VPL> : full ? route_kernel<T, VPL, true> : route_kernel<T, VPL, false>;
  return launch_overlapped(kern, grid, dim3(256), 0, 1, stream, p);
}

template <typename T>
static int dispatch_route(const RouteArgs& p, bool backward, cudaStream_t stream) {
  const int per = (p.experts + 31) / 32;
  if (per <= 1) return launch_route<T, 1>(p, backward, stream);
  if (per <= 2) return launch_route<T, 2>(p, backward, stream);
  if (per <= 4) return launch_route<T, 4>(p, backward, stream);
  if (per <= 8) return launch_route<T, 8>(p, backward, stream);
  if (per <= 16) return launch_route<T, 16>(p, backward, stream);
  return launch_route<T, 32>(p, backward, stream);
}

static int route_checks(int dtype, int64_t tokens, int64_t experts, int64_t top_k, int scoring) {
  if (dtype < FTB_F32 || dtype > FTB_F16) return FTB_E_BAD_ARG;
  if (tokens < 0 || experts <= 0 || top_k <= 0) return FTB_E_BAD_ARG;
  if (scoring != FTB_SCORE_SOFTMAX && scoring != FTB_SCORE_SIGMOID) return FTB_E_BAD_ARG;
  if (experts > FTB_MAX_EXPERTS || top_k > FTB_MAX_TOP_K || tokens > (1ll << 30)) return FTB_E_TOO_LARGE;
  return FTB_OK;
}

static int run_route(int dtype, RouteArgs& p, bool backward, cudaStream_t stream) {
  const int rc = device_ok();
  if (rc) return rc;
  const int esize = dtype == FTB_F32 ? 4 : 2;
  p.vec = (p.experts * esize) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.logits) & 15) == 0 &&
          (!backward || (reinterpret_cast<uintptr_t>(p.dlogits) & 15) == 0);
  if (dtype == FTB_F32) return dispatch_route<float>(p, backward, stream);
  if (dtype == FTB_BF16) return dispatch_route<__nv_bfloat16>(p, backward, stream);
  return dispatch_route<__half>(p, backward, stream);
}

}  // namespace ftb

extern "C" {

int ftb_route_experts(int dtype, const void* logits, const float* bias, int32_t* ids, float* weights, int64_t tokens,
                      int64_t experts, int64_t top_k, int scoring, int groups, int top_groups, int renormalize,
                      float scale, void* stream) {
  using namespace ftb;
  const int rc = route_checks(dtype, tokens, experts, top_k, scoring);
  if (rc) return rc;
  if (groups < 1 || top_groups < 1 || top_groups > groups || experts % groups != 0) return FTB_E_BAD_ARG;
  if (groups > kMaxGroups) return FTB_E_TOO_LARGE;
  if (top_k > experts / groups * top_groups) return FTB_E_BAD_ARG;
  if (tokens == 0) return FTB_OK;
  if (!logits || !ids || !weights) return FTB_E_BAD_ARG;
  RouteArgs p;
  memset(&p, 0, sizeof(p));
  p.logits = logits;
  p.bias = bias;
  p.ids = ids;
  p.weights = weights;
  p.tokens = tokens;
  p.experts = static_cast<int>(experts);
  p.top_k = static_cast<int>(top_k);
  p.scoring = scoring;
  p.groups = groups;
  p.top_groups = top_groups;
  p.renorm = renormalize != 0;
  p.scale = scale;
  int vpl = 1;  // experts per lane, as run_route picks it
  while (vpl * 32 < experts) vpl *= 2;
  const int lanes = static_cast<int>(experts / groups) / vpl;
  p.group_lanes = (experts / groups) % vpl == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  return run_route(dtype, p, false, static_cast<cudaStream_t>(stream));
}

int ftb_route_experts_backward(int dtype, const void* logits, const int32_t* ids, const float* dweights, void* dlogits,
                               int64_t tokens, int64_t experts, int64_t top_k, int scoring, int renormalize, float scale,
                               void* stream) {
  using namespace ftb;
  const int rc = route_checks(dtype, tokens, experts, top_k, scoring);
  if (rc) return rc;
  if (tokens == 0) return FTB_OK;
  if (!logits || !ids || !dweights || !dlogits) return FTB_E_BAD_ARG;
  RouteArgs p;
  memset(&p, 0, sizeof(p));
  p.logits = logits;
  p.ids = const_cast<int32_t*>(ids);
  p.dweights = dweights;
  p.dlogits = dlogits;
  p.tokens = tokens;
  p.experts = static_cast<int>(experts);
  p.top_k = static_cast<int>(top_k);
  p.scoring = scoring;
  p.groups = 1;
  p.top_groups = 1;
  p.renorm = renormalize != 0;
  p.scale = scale;
  return run_route(dtype, p, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
