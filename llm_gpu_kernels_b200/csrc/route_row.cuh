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
// Precision: the weights are FP32. The CHOICE is that of FP64, which is that of exact arithmetic unless two c, or two
// groups, are closer than a few 2^-53 of their size: where c comes from exp() in FP32, two values closer than the error
// bound of that computation could be in the wrong order. Where two neighbours of the order
// (or the groups at the border) are that close, one row in a thousand for random logits, the experts found (the two
// largest of each group) are put in order by their c in FP64, one expert per lane (exact_order, exact_groups). That is
// enough if the next expert is not close as well; otherwise the whole row is routed in FP64 (route_exact). That pass
// takes 9 us for a row, most of it instruction fetches, and a single late row shows in the call: with it alone 32768 rows
// x 256 experts took 41.5 us instead of 35.5, 4099 x 160 masked 11.5 instead of 7.5. Masks of -inf, NaN or a value below
// -1e30 cost nothing. Finite ones in between stretch the range that the FP32 keys cover, -1e9 until no key tells one real
// expert from another, and every row takes the long way: 32768 x 256 with a tenth of the logits at -1e9, softmax 123 us
// instead of 25, with groups 373 instead of 40; with a tenth of the bias there, sigmoid 132 instead of 31, with groups 274
// instead of 36.
//
// What bounds the common pass (route_fast) at many rows is the number of instructions per row, so it keeps the experts
// of a lane as sorted 32-bit keys that hold the expert too: sorting eight is 19 compare-exchanges of two integer min /
// max, each of the K rounds one maximum over the lanes and a shift of the winner's list. The K weights are computed at
// the end by K lanes at once, from logits read again, so full-precision exp and division cost one instruction sequence
// per row. Only the sum that a softmax without renormalisation divides by is that of the choice, with __expf (within
// 1.5e-6 of itself, see below): E more full exp per row would show, and the sum's own additions are as far off. 32768 rows x 256 experts FP32, sigmoid, bias, 8 groups (5.4 us would be the HBM floor): 80 us with unsorted
// keys and per-expert weights (1930 warp instructions per row), 47 us with sorted keys that leave ties and experts to
// ballots (910), 37 us like this (1018; 34.8 us if FP32 settled every row). Sixteen experts
// per lane and two rows per warp need as many instructions per row (the warp-wide redux of 32 lanes becomes four
// shuffles) and more registers: 73 us.
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
  int size;         // experts of a group (all of them without groups)
  int shift;        // log2 of the lanes of a group, see fit()
  int group_top2;   // 0: a group's value is its largest c
  int renormalize;
  int bf16_weights; // weights rounded through BF16
  float scale;
};

constexpr int kMaxGroups = 32;
constexpr float kFarBelow = -1e30f;   // c at or below it has no place of its own among a row's FP32 keys
constexpr float kSteps = 16777208.0f; // places between the smallest and the largest c: with 3 for rounding below 2^24 - 2

// Lays a row out over L lanes of P experts: a group has a power of two of whole lanes to itself, the last of them filled
// up with nothing, so that its values meet in a few shuffles. False (shift -1): the groups need more lanes than there
// are; such rows go through the general pass, experts in order. Without groups the row is one. Groups of any size
// instead of those that end at lane borders only: 8192 rows of 4 x 57 experts 10.1 instead of 41.5 us, 3 x 13 5.4 instead
// of 22.6; 1 % more for 32768 x 256.
inline bool fit(Config& cfg, int P, int L) {
  const bool grouped = cfg.kept < cfg.groups;
  cfg.shift = 0;
  while ((P << cfg.shift) < cfg.size) ++cfg.shift;
  if ((grouped ? cfg.groups : 1) << cfg.shift > L) cfg.shift = -1;
  if (!grouped) cfg.shift = 5;
  return cfg.shift >= 0;
}
// The first expert of a lane, and how many there are from it on (of which the lane holds P at most; may be negative).
template <int P, int L>
__device__ __forceinline__ void place_of(const Config& cfg, int lane, int* first, int* count) {
  if (L < 16 || cfg.shift < 0) {
    *first = lane * P;
    *count = cfg.E - lane * P;
  } else {
    const int g = lane >> cfg.shift, i = (lane & ((1 << cfg.shift) - 1)) * P;
    *first = g * cfg.size + i;
    *count = g < cfg.groups ? cfg.size - i : 0;
  }
}

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

// The L lanes of a row take part in every step together with the other rows of the warp: control flow is the same for
// the whole warp, and shuffles name all of it (a mask per row costs extra instructions at every shuffle).
constexpr unsigned kAll = 0xffffffffu;
template <int L, typename V>
__device__ __forceinline__ V sub_max(V v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
template <>
__device__ __forceinline__ uint32_t sub_max<32, uint32_t>(uint32_t v) {
  return __reduce_max_sync(kAll, v);
}
template <int L, typename V>
__device__ __forceinline__ V sub_sum(V v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
// Lanes of this row for which p holds, as the low L bits.
template <int L>
__device__ __forceinline__ unsigned sub_ballot(bool p) {
  const unsigned all = __ballot_sync(kAll, p);
  if (L == 32) return all;
  return (all >> (threadIdx.x & 31 & ~(L - 1))) & ((1u << (L & 31)) - 1u);
}

__device__ __forceinline__ int lowest_lane(unsigned lanes) { return __ffs(static_cast<int>(lanes)) - 1; }

// ids may be int32 or int64
struct Out {
  void* ids;
  float* weights;
  int wide;
  __device__ __forceinline__ void put(const Config& cfg, int slot, int e, float w) const {
    if (wide) static_cast<long long*>(ids)[slot] = e;
    else static_cast<int*>(ids)[slot] = e;
    weights[slot] = cfg.bf16_weights ? __bfloat162float(__float2bfloat16_rn(w)) : w;
  }
};

// Score of one logit; top and sum are those of the softmax (sum = 1 leaves it unnormalised). Masked logits are -inf.
__device__ __forceinline__ double score_of(const Config& cfg, double x, double top, double sum) {
  if (cfg.sigmoid) return 1.0 / (1.0 + exp(-x));                 // 0 for -inf
  return x == -INFINITY ? 0.0 : exp(x == top ? 0.0 : x - top) / sum;
}

// ------------------------------------------------------------------------------------------------ FP64, any row
// The largest 64-bit key of a row. For a whole warp two integer reductions, of the high and of the low words, are less
// than half as long as five steps of 64-bit shuffles.
template <int L>
__device__ __forceinline__ unsigned long long sub_max64(unsigned long long v) {
  if constexpr (L == 32) {
    const uint32_t hi = static_cast<uint32_t>(v >> 32), top = __reduce_max_sync(kAll, hi);
    const uint32_t low = __reduce_max_sync(kAll, hi == top ? static_cast<uint32_t>(v) : 0u);
    return static_cast<unsigned long long>(top) << 32 | low;
  } else {
    return sub_max<L>(v);
  }
}

// load(e): the logit of expert e; wanted: this row is to be written (the other rows of the warp only take part). Not
// inlined: the rare pass must not cost the common one registers. One warp in it holds up its SM's last rows, so it is
// kept short as well: sorted keys as in route_fast, whole-warp reductions.
template <int P, int L, typename Load>
__device__ __noinline__ void route_exact(const Config& cfg, const float* __restrict__ bias, int lane, bool wanted,
                                         Load load, Out out) {
  using K = Key<double>;
  using KeyT = K::type;
  const double none = -INFINITY;
  auto logit = [&](int e) { return e < cfg.E ? fmaxf(load(e), -INFINITY) : -INFINITY; };   // NaN -> -inf
  double v[P];
#pragma unroll
  for (int j = 0; j < P; ++j) v[j] = logit(lane * P + j);
  double top = none, sum = 1.0;
  if (!cfg.sigmoid) {
#pragma unroll
    for (int j = 0; j < P; ++j) top = max(top, v[j]);
    top = K::value(sub_max64<L>(K::of(top)));
    sum = 0.0;
#pragma unroll
    for (int j = 0; j < P; ++j) sum += score_of(cfg, v[j], top, 1.0);
    sum = sub_sum<L>(sum);
  }
  KeyT key[P];   // sorted, 0: not a candidate
  int place[P];  // of key[j] in the lane
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const float b = bias != nullptr && lane * P + j < cfg.E ? bias[lane * P + j] : 0.0f;
    // + 0: zeros of both signs tie
    const double c = bias != nullptr ? score_of(cfg, v[j], top, sum) + static_cast<double>(b) : v[j] + 0.0;
    key[j] = v[j] > none && b > -INFINITY ? K::of(c) : 0ull;   // false for NaN
    place[j] = j;
  }
  if (cfg.kept < cfg.groups) {
    const int size = cfg.size;
    double mine[kMaxGroups / L];          // lane i holds the values of groups i, i + L, ...
    for (int g = 0; g < cfg.groups; ++g) {
      KeyT a = 0, b = 0;                  // the two largest of the group
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const int e = lane * P + j;
        const KeyT x = e >= g * size && e < (g + 1) * size ? key[j] : 0;
        b = max(b, min(a, x));
        a = max(a, x);
      }
      const KeyT first = sub_max64<L>(a);
      const unsigned holder = sub_ballot<L>(a == first);   // its lowest lane gives up its largest
      const KeyT second = sub_max64<L>(lane == lowest_lane(holder) ? b : a);
      double value = none;
      if (first) {
        value = K::value(first);
        if (cfg.group_top2) {
          const bool scores = bias == nullptr;   // c is the score then, the keys are logits
          if (scores) value = score_of(cfg, value, top, sum);
          if (second) value += scores ? score_of(cfg, K::value(second), top, sum) : K::value(second);
        }
      }
#pragma unroll
      for (int i = 0; i < kMaxGroups / L; ++i)
        if (g == lane + i * L) mine[i] = value;
    }
    unsigned kept_groups = 0;
    for (int g = 0; g < cfg.groups; ++g) {
      double value = 0;
#pragma unroll
      for (int i = 0; i < kMaxGroups / L; ++i)
        if (g / L == i) value = mine[i];
      value = __shfl_sync(kAll, value, g & (L - 1), L);
      int before = 0;                     // groups ordered before g
#pragma unroll
      for (int i = 0; i < kMaxGroups / L; ++i) {
        const int other = lane + i * L;
        before += __popc(sub_ballot<L>(other < cfg.groups && (mine[i] > value || (mine[i] == value && other < g))));
      }
      kept_groups |= before < cfg.kept ? 1u << g : 0u;
    }
#pragma unroll
    for (int j = 0; j < P; ++j)
      if (key[j] && !(kept_groups >> ((lane * P + j) / size) & 1u)) key[j] = 0;
  }
  // descending, equal keys in the order of their places
#pragma unroll
  for (int r = 0; r < P; ++r)
#pragma unroll
    for (int i = r & 1; i + 1 < P; i += 2) {
      if (key[i] < key[i + 1]) {
        const KeyT k = key[i];
        key[i] = key[i + 1];
        key[i + 1] = k;
        const int q = place[i];
        place[i] = place[i + 1];
        place[i + 1] = q;
      }
    }
  int expert = 0;                         // lane k: the expert of slot k
  bool filled = false;
  unsigned chosen = 0;                    // of this lane's experts
  for (int k = 0; k < cfg.K; ++k) {
    const KeyT winner = sub_max64<L>(key[0]);
    const bool empty = winner == 0;       // nobody left: the lowest index not chosen yet, with weight 0
    int mine = place[0];
    if (empty) mine = __ffs(static_cast<int>(~chosen)) - 1;
    const bool holds = empty ? mine < P && lane * P + mine < cfg.E : key[0] == winner;
    const int owner = lowest_lane(sub_ballot<L>(holds));   // the lowest lane holds the lowest index
    const int at = __shfl_sync(kAll, mine, owner, L);
    if (lane == k) {
      expert = owner * P + at;
      filled = !empty;
    }
    if (lane == owner) {
      chosen |= 1u << at;
#pragma unroll
      for (int j = 0; j + 1 < P; ++j) {
        key[j] = key[j + 1];
        place[j] = place[j + 1];
      }
      key[P - 1] = 0;
    }
  }
  double w = lane < cfg.K && filled ? score_of(cfg, logit(expert), top, sum) : 0.0;
  if (cfg.renormalize) {
    const double total = sub_sum<L>(w);
    w = total > 0 ? w / total : 0.0;
  }
  if (wanted && lane < cfg.K) out.put(cfg, lane, expert, static_cast<float>(w * static_cast<double>(cfg.scale)));
}

// ------------------------------------------------------------------------------------------------ FP32
__device__ __forceinline__ void exchange(uint32_t& a, uint32_t& b) {
  const uint32_t hi = max(a, b);
  b = min(a, b);
  a = hi;
}
// Descending, by Batcher's odd-even merge network for 8 of which the exchanges beyond P fall away (a missing element
// would be smaller than any other and stay at the end).
template <int P>
__device__ __forceinline__ void sort_keys(uint32_t (&k)[P]) {
#pragma unroll
  for (int p = 1; p < 8; p *= 2)
#pragma unroll
    for (int d = p; d >= 1; d /= 2)
#pragma unroll
      for (int j = d % p; j + d < 8; j += 2 * d)
#pragma unroll
        for (int i = 0; i < d; ++i)
          if (i + j + d < P && (i + j) / (2 * p) == (i + j + d) / (2 * p)) exchange(k[i + j], k[i + j + d]);
}

// c (by_score: the score) of one expert per lane in FP64, as route_exact has it. One small function for every place that
// needs it, and no loop unrolled: the rare pass runs out of a cold instruction cache.
template <int P, int L, typename Load>
__device__ __noinline__ double exact_choice(const Config& cfg, const float* __restrict__ bias, int lane, int expert,
                                            bool by_score, Load load) {
  auto logit = [&](int e) { return e < cfg.E ? fmaxf(load(e), -INFINITY) : -INFINITY; };   // NaN -> -inf
  const double x = logit(expert);
  if (bias == nullptr && !by_score) return x + 0.0;
  double top = -INFINITY, sum = 1.0;
  if (!cfg.sigmoid) {
    float high = -INFINITY;
#pragma unroll 1
    for (int j = 0; j < P; ++j) high = fmaxf(high, logit(lane * P + j));
    top = Key<float>::value(sub_max<L>(Key<float>::of(high)));
    sum = 0.0;
#pragma unroll 1
    for (int j = 0; j < P; ++j) sum += score_of(cfg, logit(lane * P + j), top, 1.0);
    sum = sub_sum<L>(sum);
  }
  const double s = score_of(cfg, x, top, sum);
  return bias != nullptr && expert < cfg.E ? s + static_cast<double>(bias[expert]) : s;
}

// Whether the group of this lane is kept, decided in FP64. a, second: the two largest keys of the lane's group of
// `lanes` lanes.
template <int P, int L, typename Load>
__device__ __noinline__ bool exact_groups(const Config& cfg, const float* __restrict__ bias, int lane, int lanes,
                                          uint32_t a, uint32_t second, bool by_score, Load load) {
  const double va = exact_choice<P, L>(cfg, bias, lane, 255 - (a & 255u), by_score, load);
  const double vb = exact_choice<P, L>(cfg, bias, lane, 255 - (second & 255u), by_score, load);
  double value = a ? va : -INFINITY;
  if (second) value = cfg.group_top2 ? va + vb : max(va, vb);
  int before = 0;
#pragma unroll 1
  for (int g = 0; g < cfg.groups; ++g) {
    const double v = __shfl_sync(kAll, value, g * lanes, L);
    before += v > value || (v == value && (g + 1) * lanes <= lane);
  }
  return before < cfg.kept;
}

// The candidates of lanes 0 .. K in the order of FP64; lane k gets the k-th.
template <int P, int L, typename Load>
__device__ __noinline__ uint32_t exact_order(const Config& cfg, const float* __restrict__ bias, int lane, uint32_t won,
                                             Load load) {
  const int expert = 255 - static_cast<int>(won & 255u);
  const double c = exact_choice<P, L>(cfg, bias, lane, expert, false, load);
  int before = 0;
#pragma unroll 1
  for (int i = 0; i <= cfg.K; ++i) {
    const double v = __shfl_sync(kAll, c, i, L);
    const uint32_t other = __shfl_sync(kAll, won, i, L);
    before += other != 0 && (won == 0 || v > c || (v == c && 255 - static_cast<int>(other & 255u) < expert));
  }
  uint32_t mine = 0;
#pragma unroll 1
  for (int i = 0; i <= cfg.K; ++i) {
    const uint32_t other = __shfl_sync(kAll, won, i, L);
    if (__shfl_sync(kAll, before, i, L) == lane && other != 0) mine = other;
  }
  return mine;
}

// Lane n .. K-1: the (lane - n)-th lowest index that is not among the experts of lanes 0 .. n-1. Starting from that rank,
// an index moves up by the chosen ones at or below it until it stays. (Left to route_exact, 8192 rows of 128 experts with
// nine in ten masked took 36 us instead of 9.4.)
template <int L>
__device__ __noinline__ int fill_slot(int K, int lane, int n, int expert) {
  int e = lane - n;
  bool moved = true;
#pragma unroll 1
  while (moved) {
    int below = 0;
#pragma unroll 1
    for (int i = 0; i < K; ++i) {
      const int chosen = __shfl_sync(kAll, expert, i, L);
      below += i < n && chosen <= e;
    }
    const int at = lane - n + below;
    moved = __any_sync(kAll, lane >= n && lane < K && at != e);
    e = at;
  }
  return e;
}

// Returns false when FP32 and a look at the candidates in FP64 cannot settle the row; otherwise slot `lane` < K of the
// row is `expert` with weight `w`.
// l[j]: logits of experts first + j (-inf: none), b[j]: biases.
//
// Keys are (q << 8) | (255 - expert): the larger key has the larger q, or the lower index at equal q, so every key is
// different, the winner of a round names its expert and no tie needs a second look. q has 24 bits and is at least 1
// (key 0: not a candidate). Logits of 16 bits without a bias give their leading 24 bits, which are exact. Everything
// else gives its place between the smallest and the largest c of the row: q = 2 + (c - base) * scale, monotonic in c and
// off by less than 2 from rounding. Values of -1e30 and less, the lowest finite ones that programs mask experts with,
// stay out of that range and are all q = 1: behind every other expert, in an order that only FP64 knows.
template <int P, int L, typename Load>
__device__ __forceinline__ bool route_fast(const Config& cfg, float (&l)[P], const float (&b)[P], int lane, int first,
                                           const float* __restrict__ bias, Load load, int* expert, float* weight) {
  using K = Key<float>;
  const bool biased = bias != nullptr;
  const float none = -INFINITY;
  const bool grouped = L >= 16 && cfg.kept < cfg.groups;   // fewer lanes route without groups only (route.cu)
  float top = none;
  uint32_t low_bits = 0;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    l[j] = fmaxf(l[j], none);   // NaN -> -inf
    low_bits |= __float_as_uint(l[j]);
    top = fmaxf(top, l[j]);
  }
  top = K::value(sub_max<L>(K::of(top)));
  float unit = 1.0f, sum = 1.0f;   // unit: the largest score there can be
  if (!cfg.sigmoid && (biased || grouped || !cfg.renormalize)) {
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j) sum += l[j] > none ? __expf(l[j] == top ? 0.0f : l[j] - top) : 0.0f;
    sum = sub_sum<L>(sum);
    unit = __fdividef(1.0f, sum);
  }
  auto score = [&](float x) {   // approximate; for the choice only
    return cfg.sigmoid ? __fdividef(1.0f, 1.0f + __expf(-x)) : unit * __expf(x == top ? 0.0f : x - top);
  };
  // Without a bias c is the logit; 16-bit logits, even as FP32, have nothing in their last 8 bits. One answer for the
  // warp: the rows it routes are of one tensor.
  const bool exact = !biased && __all_sync(kAll, (low_bits & 255u) == 0);
  float c[P];
#pragma unroll
  for (int j = 0; j < P; ++j) c[j] = l[j];
  if (biased) {
    if (cfg.sigmoid) {
#pragma unroll
      for (int j = 0; j < P; ++j) c[j] = fmaxf(l[j] > none ? __fdividef(1.0f, 1.0f + __expf(-l[j])) + b[j] : none, none);
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) c[j] = fmaxf(l[j] > none ? unit * __expf(l[j] == top ? 0.0f : l[j] - top) + b[j] : none, none);
    }
  }
  uint32_t key[P];
  float base = 0.0f, step = 0.0f;    // c = base + (q - 2) * step, about
  uint32_t unsure = 0;               // two q this close or closer may be in the wrong order
  bool close = false;
  bool vague = false;                // the keys do not tell what groups are worth
  if (exact) {
#pragma unroll
    for (int j = 0; j < P; ++j)   // + 0: zeros of both signs tie
      key[j] = c[j] > none ? (K::of(c[j] + 0.0f) & ~255u) | (255u - (first + j)) : 0u;
  } else {
    float low = INFINITY, high = none;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      low = fminf(low, c[j] > kFarBelow ? c[j] : INFINITY);
      high = fmaxf(high, c[j]);
    }
    if (biased) high = K::value(sub_max<L>(K::of(high)));
    else high = top;
    low = -K::value(sub_max<L>(K::of(-low)));
    low = fminf(low, high);
    const float range = high - low;
    // a row of one value, or with an infinity: every q is the same, which settles nothing
    const float scale = range > 1e-30f && range < INFINITY ? kSteps / range : 0.0f;
    base = low;
    step = scale > 0.0f ? range / kSteps : 0.0f;
    const float least = scale > 0.0f ? -1.0f : 0.0f;   // for c below `low`
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const float q = fmaxf(least, (c[j] - low) * scale) + 2.0f;   // NaN (infinities): scale is 0, q 2
      key[j] = c[j] > none ? __float2uint_rn(q) << 8 | (255u - (first + j)) : 0u;
    }
    // The error of c: __expf is within 2^-22 + |x| 2^-23, which moves a sigmoid by a quarter of that and a softmax score
    // by its own size times it (|x| exp(x) <= 0.37); a reciprocal of 2^-23; up to 13 additions of a softmax sum (8 in a
    // lane, 5 levels of the tree): 4e-7 for a sigmoid, 1.5e-6 of the largest score for a softmax, and half an ulp of c.
    if (biased) {
      const float widest = fmaxf(fabsf(low), fabsf(high));
      unsure = static_cast<uint32_t>(fminf(2.0f * ((cfg.sigmoid ? 4e-7f : 1.5e-6f * unit) + 6e-8f * widest) * scale + 5.0f, 16777215.0f));
    }
    // Scores are compared by logits a step or two off, so a step has to be small. A sum with a c far below is taken for
    // less than any two other c, which holds while these are not of its size.
    vague = scale == 0.0f || (cfg.group_top2 && (biased ? !(2.0f * low > high + kFarBelow) : step > 0.1f));
  }
  sort_keys<P>(key);
  if (grouped) {
    const int lanes = 1 << cfg.shift;
    uint32_t a = key[0], second = P > 1 ? key[P > 1] : 0u;
    for (int o = 1; o < lanes; o <<= 1) {
      const uint32_t oa = __shfl_xor_sync(kAll, a, o), ob = __shfl_xor_sync(kAll, second, o);
      second = max(min(a, oa), max(second, ob));
      a = max(a, oa);
    }
    auto value_of = [&](uint32_t k) {
      // the last 8 bits of an exact logit are zeros: in the key of a negative one, which is inverted, they are ones
      return exact ? K::value(k >> 31 ? k & ~255u : k | 255u) : base + static_cast<float>(static_cast<int>(k >> 8) - 2) * step;
    };
    auto far_below = [](uint32_t k) { return k < 512u; };   // q = 1; exact keys are larger
    const bool by_score = cfg.group_top2 && !biased;
    // Far below: the score is 0, and so it is in FP64, at more than 1e22 under the largest logit (or 1e30 under 0). A c
    // there is unknown, and so is a sum with it: such groups tie with each other and come before those that have nobody.
    constexpr float kUnknown = -3e38f;
    float value = none;
    if (a) {
      if (by_score) {
        value = far_below(a) ? 0.0f : score(value_of(a));
        if (second) value += far_below(second) ? 0.0f : score(value_of(second));
      } else if (cfg.group_top2 && second) {
        value = far_below(second) ? kUnknown : value_of(a) + value_of(second);
      } else {
        value = far_below(a) ? kUnknown : value_of(a);
      }
    }
    const int leader = lane & ~(lanes - 1);   // of this lane's group
    uint32_t group_key = lane == leader && lane >> cfg.shift < cfg.groups ? K::of(value) : 0u;
    bool kept = false;
    uint32_t last = 0;
    for (int g = 0; g < cfg.kept; ++g) {
      last = sub_max<L>(group_key);
      const int winner = lowest_lane(sub_ballot<L>(group_key == last));
      kept |= leader == winner;
      if (lane == winner) group_key = 0u;
    }
    if (!exact || by_score) {   // is the border between the kept groups and the others certain?
      const float border = K::value(last), next = K::value(sub_max<L>(group_key));
      // two values of two c each (or scores, whose logits are off by `step`)
      const float far = by_score ? 4.0f * (2e-6f * unit + step) : 2.0f * step * static_cast<float>(unsure + 2u) + 2.4e-7f * fabsf(border);
      close = vague || border - next <= far;   // infinities compare false
      if (__any_sync(kAll, close)) {
        // In FP64 from the two largest of each group. They have to be certain: no third one close to the second.
        int near = 0;
#pragma unroll
        for (int j = 0; j < P; ++j) near += key[j] != 0 && (exact ? key[j] >= second : (key[j] >> 8) + unsure >= second >> 8);
        for (int o = 1; o < lanes; o <<= 1) near += __shfl_xor_sync(kAll, near, o);
        const bool certain = sub_ballot<L>(near > 2) == 0;
        const bool exactly = exact_groups<P, L>(cfg, bias, lane, lanes, a, second, by_score, load);
        if (close) kept = exactly;
        close = close && !certain;
      }
    }
    if (!kept) {
#pragma unroll
      for (int j = 0; j < P; ++j) key[j] = 0u;
    }
  }
  // K rounds, and one more where the border matters; sub-lane k keeps the winner of round k
  uint32_t won = 0, next = 0;
  const int rounds = exact ? cfg.K : cfg.K + 1;
  for (int k = 0; k < rounds; ++k) {
    const uint32_t winner = sub_max<L>(key[0]);
    if (lane == k) won = winner;
    if (lane == k - 1) next = winner;
    if (key[0] == winner) {
#pragma unroll
      for (int j = 0; j + 1 < P; ++j) key[j] = key[j + 1];
      key[P - 1] = 0u;
    }
  }
  if (!exact) {
    const bool tight = lane < cfg.K && next && (won >> 8) - (next >> 8) <= unsure;
    if (__any_sync(kAll, tight)) {
      // In FP64 among the K + 1 found, if they are certain: the one after them is not close to the last.
      const uint32_t after = sub_max<L>(key[0]);
      const unsigned uncertain = sub_ballot<L>(cfg.K >= L || (lane == cfg.K && after && (won >> 8) - (after >> 8) <= unsure));
      const uint32_t order = exact_order<P, L>(cfg, bias, lane, won, load);
      if (uncertain == 0) won = order;
      else close |= tight;
    }
  }
  const bool empty = lane < cfg.K && won == 0;
  const unsigned unfilled = sub_ballot<L>(empty);
  const bool nothing = (unfilled & 1u) != 0;   // a row whose mask leaves nothing: the lowest indices with weight 0
  const unsigned undecided = sub_ballot<L>(close);   // by every lane: not behind a condition that rows differ in
  bool settled = nothing || undecided == 0;
  *expert = nothing ? lane : static_cast<int>(255u - (won & 255u));
  const bool partly = unfilled != 0 && !nothing;   // fewer experts left than slots
  if (L == 32 ? partly : __any_sync(kAll, partly)) {
    const int filler = fill_slot<L>(cfg.K, lane, cfg.K - __popc(unfilled), *expert);
    if (empty) *expert = filler;
  }
  float w = 0.0f;
  if (lane < cfg.K && settled && !empty) {
    const float x = load(*expert);
    w = cfg.sigmoid ? 1.0f / (1.0f + expf(-x)) : expf(x == top ? 0.0f : x - top);
  }
  if (cfg.renormalize) {
    const float total = sub_sum<L>(w);
    settled = settled && (nothing || total >= 1e-30f);   // scores below that have lost their ratio in FP32
    w = nothing ? 0.0f : w / total;
  } else if (!cfg.sigmoid) {
    w = nothing ? 0.0f : w / sum;
  }
  *weight = w * cfg.scale;
  return settled;
}

// Routes the rows of a warp, 32 / L of them: lane (0..L-1 of its row's lanes) holds logits and biases of the experts
// that place_of gives it; load(e) gives a logit of the row again. The whole warp calls it; rows that are not `live`
// (their lanes hold any logits, and load() is called for them) are not written. P * L >= E, L >= K.
template <int P, int L, typename Load>
__device__ __forceinline__ void route_row(const Config& cfg, float (&l)[P], const float (&b)[P],
                                          const float* __restrict__ bias, int lane, bool live, Load load,
                                          Out out) {
  bool settled = false;
  if (L < 16 || cfg.shift >= 0) {
    int expert, first, count;
    float w;
    place_of<P, L>(cfg, lane, &first, &count);
    settled = route_fast<P, L>(cfg, l, b, lane, first, bias, load, &expert, &w);
    if (live && settled && lane < cfg.K) out.put(cfg, lane, expert, w);
  }
  if (__any_sync(kAll, live && !settled)) route_exact<P, L>(cfg, bias, lane, live && !settled, load, out);
}

// A lane's logits and biases, one by one.
template <int P, int L, typename Load>
__device__ __forceinline__ void load_row(const Config& cfg, const float* __restrict__ bias, int lane, const Load& load,
                                         float (&l)[P], float (&b)[P]) {
  int first, count;
  place_of<P, L>(cfg, lane, &first, &count);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    l[j] = j < count ? load(first + j) : -INFINITY;
    b[j] = bias != nullptr && j < count ? bias[first + j] : 0.0f;
  }
}

}  // namespace route
}  // namespace b200moe
