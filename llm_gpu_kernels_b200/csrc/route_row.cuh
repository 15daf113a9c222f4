// Routing of one token by the lanes of a (sub-)warp: scores, balance bias, expert groups, top-k, weights.
// Shared by the operator on given logits (route.cu) and by the two routers that compute the logits themselves
// (router_tc.cu, router.cu).
//
//   s_e = softmax over the E logits, or 1 / (1 + exp(-l_e))
//   c_e = s_e + bias_e; without a bias the choice goes by l_e itself, which orders the experts as s_e does
//   groups of E / G consecutive experts, valued by their largest c or by the sum of their two largest c (of s without
//   a bias); only the `kept` groups of the largest values take part
//   ids = the K experts of largest c, in that order; ties, here and among groups, go to the lower index
//   w = s at those experts, divided by their sum if asked for, times `scale`
// An expert whose logit (or bias) is NaN or -inf is masked: no score, never chosen while another is left. Slots that
// nobody can fill get the lowest indices not chosen yet, with weight 0, so the ids stay valid for the dispatch.
//
// Precision: the weights are FP32. The CHOICE is that of exact arithmetic: where c comes from exp() in FP32, two
// values closer than the error bound of that computation could be in the wrong order, so a row in which two
// neighbours of the order (or the groups at the border) are that close is routed again in FP64. That is one row in
// about a thousand for random logits and costs nothing measurable; an FP64 pass for every row would take the
// 32768 x 256 case from HBM-bound to several times its time.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace b200moe {
namespace route {

struct Config {
  int E, K;
  int sigmoid;      // 0: softmax scores
  int groups, kept; // groups = 1: no groups
  int group_top2;   // 0: a group's value is its largest c
  int renormalize;
  int bf16_weights; // weights rounded through BF16
  float scale;
};

constexpr int kMaxGroups = 32;
// |c_fp32 - c| <= kScoreError * max(1, |c|): expf within 2 ulp, 13 additions of the softmax sum (up to 8 per lane and
// 5 levels of the tree), one division and the bias addition are below 17 half-ulps = 1.1e-6; rounded up.
constexpr float kScoreError = 1.5e-6f;

template <typename F> struct Key;
template <> struct Key<float> {
  using type = uint32_t;
  static __device__ __forceinline__ type of(float v) {
    const uint32_t u = __float_as_uint(v);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);   // unsigned order = float order; -inf -> 0x007fffff > 0
  }
  static __device__ __forceinline__ float value(type k) {
    return __uint_as_float((k >> 31) ? (k ^ 0x80000000u) : ~k);
  }
};
template <> struct Key<double> {
  using type = unsigned long long;
  static __device__ __forceinline__ type of(double v) {
    const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v));
    return u ^ ((u >> 63) ? ~0ull : 0x8000000000000000ull);
  }
  static __device__ __forceinline__ double value(type k) {
    return __longlong_as_double(static_cast<long long>((k >> 63) ? (k ^ 0x8000000000000000ull) : ~k));
  }
};

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

template <int L, typename V>
__device__ __forceinline__ V sub_max(V v, unsigned mask) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(mask, v, o));
  return v;
}
template <>
__device__ __forceinline__ uint32_t sub_max<32, uint32_t>(uint32_t v, unsigned) {
  return __reduce_max_sync(0xffffffffu, v);
}
template <int L, typename V>
__device__ __forceinline__ V sub_sum(V v, unsigned mask) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  return v;
}

template <typename F>
__device__ __forceinline__ F minus_inf() { return static_cast<F>(-INFINITY); }

// Which of this lane's experts may be chosen after the group step: bit j. `v` holds c (or the logit) of the
// candidates of `ok`, `s` the scores. Full warp (L = 32). Sets *close when FP32 cannot decide the border.
template <typename F, int P>
__device__ __forceinline__ unsigned keep_groups(const Config& cfg, const F (&v)[P], const F (&s)[P], unsigned ok,
                                                int lane, bool by_score, bool inexact, bool* close) {
  const int size = cfg.E / cfg.groups;
  const F none = minus_inf<F>();
  F mine = none;                          // lane g: value of group g
  const int lanes = size / P;             // lanes per group where groups end at lane borders
  if (size % P == 0 && (lanes & (lanes - 1)) == 0) {
    F a = none, b = none;                 // the two largest of this lane, then of its group
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const F x = (ok >> j & 1u) ? (by_score ? s[j] : v[j]) : none;
      b = max(b, min(a, x));
      a = max(a, x);
    }
    for (int o = 1; o < lanes; o <<= 1) {
      const F oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
      b = max(min(a, oa), max(b, ob));
      a = max(a, oa);
    }
    const F value = cfg.group_top2 && b != none ? a + b : a;
    mine = __shfl_sync(0xffffffffu, value, (lane * lanes) & 31);
    if (lane >= cfg.groups) mine = none;
  } else {
    for (int g = 0; g < cfg.groups; ++g) {
      F a = none, b = none;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int e = lane * P + j;
        const F x = (ok >> j & 1u) && e >= g * size && e < (g + 1) * size ? (by_score ? s[j] : v[j]) : none;
        b = max(b, min(a, x));
        a = max(a, x);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const F oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
        b = max(min(a, oa), max(b, ob));
        a = max(a, oa);
      }
      if (lane == g) mine = cfg.group_top2 && b != none ? a + b : a;
    }
  }
  int before = 0;                         // groups ordered before this lane's
  for (int g = 0; g < cfg.groups; ++g) {
    const F other = __shfl_sync(0xffffffffu, mine, g);
    before += other > mine || (other == mine && g < lane) ? 1 : 0;
  }
  const bool in = lane < cfg.groups, kept = in && before < cfg.kept;
  if (inexact) {
    F low = kept ? mine : static_cast<F>(INFINITY), high = in && !kept ? mine : none;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      low = min(low, __shfl_xor_sync(0xffffffffu, low, o));
      high = max(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    F size_of = 1;   // the error of a value goes by the c it is made of, not by their sum
#pragma unroll
    for (int j = 0; j < P; ++j)
      if (ok >> j & 1u) size_of = max(size_of, abs(v[j]));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) size_of = max(size_of, __shfl_xor_sync(0xffffffffu, size_of, o));
    // each value is a sum of up to two c; infinities compare false
    if (low - high <= static_cast<F>(4 * kScoreError) * size_of) *close = true;
  }
  const unsigned groups = __ballot_sync(0xffffffffu, kept);
  unsigned keep = 0;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int e = lane * P + j;
    if (e < cfg.E && (groups >> (e / size) & 1u)) keep |= 1u << j;
  }
  return keep;
}

// One pass in precision F. Returns false when (F = float) two values are too close for it.
template <typename F, int P, int L, typename IdT>
__device__ bool route_pass(const Config& cfg, const float (&l)[P], const float* __restrict__ bias, int lane,
                           unsigned mask, IdT* __restrict__ ids, float* __restrict__ weights) {
  using K = Key<F>;
  using KeyT = typename K::type;
  constexpr bool kFast = sizeof(F) == 4;
  const F none = minus_inf<F>();
  unsigned ok = 0;
  F v[P], s[P];
  F top = none;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int e = lane * P + j;
    v[j] = static_cast<F>(l[j]);
    if (e < cfg.E && l[j] > -INFINITY) {   // false for NaN
      ok |= 1u << j;
      top = max(top, v[j]);
    }
  }
  const bool by_score = cfg.groups > 1 && cfg.group_top2 && bias == nullptr;   // group values only
  const bool scores_first = bias != nullptr || by_score;
  if (!cfg.sigmoid) {
    top = sub_max<L>(top, mask);
    F sum = 0;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      s[j] = (ok >> j & 1u) ? exp_of(v[j] == top ? static_cast<F>(0) : v[j] - top) : static_cast<F>(0);
      sum += s[j];
    }
    if (scores_first || !cfg.renormalize) {   // otherwise the sum cancels
      sum = sub_sum<L>(sum, mask);
#pragma unroll
      for (int j = 0; j < P; ++j) s[j] = (ok >> j & 1u) ? s[j] / sum : static_cast<F>(0);
    }
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j) s[j] = (ok >> j & 1u) ? 1 / (1 + exp_of(-v[j])) : static_cast<F>(0);
  }
  if (bias != nullptr) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int e = lane * P + j;
      const float b = e < cfg.E ? bias[e] : 0.0f;
      v[j] = s[j] + static_cast<F>(b);
      if (!(b > -INFINITY)) ok &= ~(1u << j);
    }
  }
  bool close = false;
  if (L == 32 && cfg.groups > 1) ok &= keep_groups<F, P>(cfg, v, s, ok, lane, by_score, kFast && scores_first, &close);
  KeyT key[P];
  int rank[P];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    key[j] = (ok >> j & 1u) ? K::of(v[j]) : static_cast<KeyT>(0);   // 0: not a candidate
    rank[j] = -1;
  }
  const bool check = kFast && bias != nullptr;
  KeyT last = 0;
  F total = 0;
  for (int k = 0; k < cfg.K; ++k) {
    KeyT best = key[0];
#pragma unroll
    for (int j = 1; j < P; ++j) best = max(best, key[j]);
    const KeyT winner = sub_max<L>(best, mask);
    if (winner == 0) {                       // nobody left: the lowest indices not chosen, weight 0
      for (; k < cfg.K; ++k) {
        int e = 0x7fffffff;
#pragma unroll
        for (int j = P - 1; j >= 0; --j)
          if (rank[j] < 0 && lane * P + j < cfg.E) e = lane * P + j;
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) e = min(e, __shfl_xor_sync(mask, e, o));
#pragma unroll
        for (int j = 0; j < P; ++j)
          if (lane * P + j == e) { rank[j] = k; s[j] = 0; }
      }
      break;
    }
    if (check && k > 0) {
      const F a = K::value(last), b = K::value(winner);
      if (a - b <= static_cast<F>(2 * kScoreError) * max(static_cast<F>(1), abs(a))) close = true;
    }
    last = winner;
    const unsigned holders = __ballot_sync(mask, best == winner) & mask;
    bool mine = (holders & (0u - holders)) == 1u << (threadIdx.x & 31);   // the lowest lane holds the lowest index
#pragma unroll
    for (int j = 0; j < P; ++j) {
      if (mine && key[j] == winner) {
        key[j] = 0;
        rank[j] = k;
        total += s[j];
        mine = false;
      }
    }
  }
  if (check) {   // the first expert left out
    KeyT best = key[0];
#pragma unroll
    for (int j = 1; j < P; ++j) best = max(best, key[j]);
    best = sub_max<L>(best, mask);
    const F a = K::value(last), b = K::value(best);
    if (best != 0 && a - b <= static_cast<F>(2 * kScoreError) * max(static_cast<F>(1), abs(a))) close = true;
  }
  if (close) return false;
  if (cfg.renormalize) {
    total = sub_sum<L>(total, mask);
    if (kFast && !(total >= static_cast<F>(1e-30))) return false;   // scores this small have lost their ratio in FP32
  }
  const F factor = static_cast<F>(cfg.scale);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    if (rank[j] >= 0) {
      F w = s[j];
      if (cfg.renormalize) w = total > 0 ? w / total : static_cast<F>(0);
      float r = static_cast<float>(w * factor);
      if (cfg.bf16_weights) r = __bfloat162float(__float2bfloat16_rn(r));
      ids[rank[j]] = static_cast<IdT>(lane * P + j);
      weights[rank[j]] = r;
    }
  }
  return true;
}

// Not inlined: the rare pass must not cost the common one registers.
template <int P, int L, typename IdT>
__device__ __noinline__ void route_again(const Config& cfg, const float (&l)[P], const float* __restrict__ bias, int lane,
                                         unsigned mask, IdT* __restrict__ ids, float* __restrict__ weights) {
  route_pass<double, P, L, IdT>(cfg, l, bias, lane, mask, ids, weights);
}

// Routes one row: lane (0..L-1 of the row's lanes, which are the lanes of `mask`) holds the logits of experts
// lane*P .. lane*P+P-1 in l; ids / weights point at the row's K entries. P * L >= E; groups > 1 needs L = 32.
template <int P, int L, typename IdT>
__device__ __forceinline__ void route_row(const Config& cfg, const float (&l)[P], const float* __restrict__ bias, int lane,
                                          unsigned mask, IdT* __restrict__ ids, float* __restrict__ weights) {
  if (!route_pass<float, P, L, IdT>(cfg, l, bias, lane, mask, ids, weights))
    route_again<P, L, IdT>(cfg, l, bias, lane, mask, ids, weights);
}

}  // namespace route
}  // namespace b200moe
