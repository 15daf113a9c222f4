// Routing on given logits: [T, E] in BF16, FP16 or FP32 (rows may be strided) to ids and weights [T, K]. The formula is
// in route_row.cuh; a row is held in registers by 32, 16, 8 or 4 lanes, up to 8 experts each, and read from HBM once.
// Bound by HBM only for long prompts (32768 x 256 FP32: 33.5 MB in, 2 MB out, floor 5.4 us); at a serving batch one
// launch is all there is.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "pdl.cuh"
#include "plan.h"
#include "route_row.cuh"

namespace b200moe {
namespace {

constexpr int kThreads = 128;

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// N floats or halves of one lane as FP32: one or two vector loads (N * sizeof(T) of 8, 16 or 32 bytes) or N scalar ones.
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* src, float (&v)[N]) {
  constexpr int kBytes = N * sizeof(T);
  union { T t[N]; uint32_t w[(kBytes + 3) / 4]; } raw;
  if constexpr (kBytes % 16 == 0) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) {
      const uint4 q = *(reinterpret_cast<const uint4*>(src) + i);
      raw.w[4 * i] = q.x; raw.w[4 * i + 1] = q.y; raw.w[4 * i + 2] = q.z; raw.w[4 * i + 3] = q.w;
    }
  } else if constexpr (kBytes == 8) {
    const uint2 q = *reinterpret_cast<const uint2*>(src);
    raw.w[0] = q.x; raw.w[1] = q.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) raw.t[i] = src[i];
  }
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = to_float(raw.t[j]);
}

// kVec: a lane's P logits, and its P biases, are each one aligned piece.
template <typename T, int P, int L, bool kVec>
__global__ void __launch_bounds__(kThreads, 8)   // 64 registers: the rare FP64 pass may spill, the common one does not
route_kernel(const T* __restrict__ logits, long long pitch, const float* __restrict__ bias, void* __restrict__ ids,
             int ids_are_int64, float* __restrict__ weights, int tokens, const __grid_constant__ route::Config cfg) {
  pdl_launch_dependents();
  pdl_wait();   // the logits may come from the kernel just before; ids / weights may still be read by it
  const int lane = threadIdx.x & (L - 1);
  const long long wanted = static_cast<long long>(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
  const bool live = wanted < tokens;
  const long long row = live ? wanted : tokens - 1;   // lanes past the end follow the last row and write nothing
  const T* row_logits = logits + row * pitch;
  float l[P], b[P];
  auto logit = [row_logits](int e) { return to_float(row_logits[e]); };
  if (kVec) {
    int e, count;
    route::place_of<P, L>(cfg, lane, &e, &count);
    const bool inside = count > 0;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      l[j] = -INFINITY;
      b[j] = 0.0f;
    }
    if (inside) load_vec(row_logits + e, l);
    if (inside && bias != nullptr) load_vec(bias + e, b);
  } else {
    route::load_row<P, L>(cfg, bias, lane, logit, l, b);
  }
  const long long first = row * cfg.K;
  const route::Out out{ids_are_int64 ? static_cast<void*>(static_cast<long long*>(ids) + first)
                                     : static_cast<void*>(static_cast<int*>(ids) + first), weights + first, ids_are_int64};
  route::route_row<P, L>(cfg, l, b, bias, lane, live, logit, out);
}

template <typename T, int P, int L>
cudaError_t launch(const B200MoeRouteArgs& a, route::Config cfg, cudaStream_t s) {
  route::fit(cfg, P, L);
  const T* logits = static_cast<const T*>(a.logits);
  auto* bias = static_cast<const float*>(a.bias);
  auto* w = static_cast<float*>(a.weights);
  constexpr bool kPow2 = (P & (P - 1)) == 0;
  const size_t piece = P * sizeof(T) < 16 ? P * sizeof(T) : 16;
  const bool vec = kPow2 && (cfg.shift < 0 ? cfg.E : cfg.size) % P == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0 &&
                   (a.pitch * sizeof(T)) % piece == 0 && reinterpret_cast<uintptr_t>(bias) % 16 == 0;
  const int rows = kThreads / L;
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(a.tokens) + rows - 1) / rows));
  const long long pitch = a.pitch;
  if constexpr (kPow2)
    if (vec)
      return launch_pdl(route_kernel<T, P, L, true>, grid, dim3(kThreads), 0, s, logits, pitch, bias, a.ids,
                        a.ids_are_int64, w, a.tokens, cfg);
  return launch_pdl(route_kernel<T, P, L, false>, grid, dim3(kThreads), 0, s, logits, pitch, bias, a.ids, a.ids_are_int64,
                    w, a.tokens, cfg);
}

// Lanes and experts per lane. Few lanes per row, so that rows share a warp (the instructions of a round are then paid
// once for several rows), but at least K: a lane per weight. With groups, the fewest experts per lane that leave every
// group a power of two of whole lanes; where even eight do not (three groups of 70, say) the kernel takes its general
// pass for every row.
template <typename T, int L>
cudaError_t launch_lanes(const B200MoeRouteArgs& a, const route::Config& cfg, cudaStream_t s) {
  const bool grouped = cfg.kept < cfg.groups;
  auto fits = [&](int p) {
    route::Config c = cfg;
    return p * L >= cfg.E && route::fit(c, p, L);
  };
  if constexpr (L >= 16)
    if (grouped && fits(1)) return launch<T, 1, L>(a, cfg, s);
  if (fits(2)) return launch<T, 2, L>(a, cfg, s);
  if constexpr (L >= 16)
    if (grouped && fits(3)) return launch<T, 3, L>(a, cfg, s);
  if (fits(4)) return launch<T, 4, L>(a, cfg, s);
  if constexpr (L >= 16) {
    if (grouped && fits(5)) return launch<T, 5, L>(a, cfg, s);
    if (grouped && fits(6)) return launch<T, 6, L>(a, cfg, s);
    if (grouped && fits(7)) return launch<T, 7, L>(a, cfg, s);
  }
  return launch<T, 8, L>(a, cfg, s);
}

template <typename T>
cudaError_t launch_typed(const B200MoeRouteArgs& a, const route::Config& cfg, cudaStream_t s) {
  if (cfg.kept == cfg.groups) {
    if (cfg.E <= 32 && cfg.K <= 4) return launch_lanes<T, 4>(a, cfg, s);
    if (cfg.E <= 64 && cfg.K <= 8) return launch_lanes<T, 8>(a, cfg, s);
  }
  route::Config half = cfg;
  if (cfg.E <= 128 && cfg.K <= 16 && route::fit(half, 8, 16)) return launch_lanes<T, 16>(a, cfg, s);
  return launch_lanes<T, 32>(a, cfg, s);
}

}  // namespace

// Host-side check of a router configuration for E experts and K slots; sets the error message.
bool route_config_ok(const B200MoeRouterConfig& c, int experts, int topk) {
  if (c.score != B200MOE_SCORE_SOFTMAX && c.score != B200MOE_SCORE_SIGMOID) {
    set_error("router: unknown score function %d", c.score);
    return false;
  }
  if (c.groups < 1 || c.groups > route::kMaxGroups || experts % c.groups || c.kept_groups < 1 || c.kept_groups > c.groups) {
    set_error("router: groups must divide the %d experts, at most %d of them, 1 <= kept_groups <= groups (got %d, %d)",
              experts, route::kMaxGroups, c.groups, c.kept_groups);
    return false;
  }
  if (c.group_score != B200MOE_GROUP_MAX && c.group_score != B200MOE_GROUP_TOP2) {
    set_error("router: unknown group score %d", c.group_score);
    return false;
  }
  if (topk < 1 || topk > 32 || topk > c.kept_groups * (experts / c.groups)) {
    set_error("router: topk must be in [1,32] and fit the experts of the kept groups (topk=%d)", topk);
    return false;
  }
  if (!(c.scale > 0.0f && c.scale <= 3.402823466e38f)) {
    set_error("router: scale must be positive and finite");
    return false;
  }
  return true;
}

route::Config route_config(const B200MoeRouterConfig& c, int experts, int topk) {
  route::Config cfg;
  cfg.E = experts;
  cfg.K = topk;
  cfg.sigmoid = c.score == B200MOE_SCORE_SIGMOID;
  cfg.groups = c.groups;
  cfg.kept = c.kept_groups;
  cfg.size = c.kept_groups < c.groups ? experts / c.groups : experts;
  cfg.shift = -1;
  cfg.group_top2 = c.group_score == B200MOE_GROUP_TOP2;
  cfg.renormalize = c.renormalize != 0;
  cfg.bf16_weights = c.bf16_weights != 0;
  cfg.scale = c.scale;
  return cfg;
}

}  // namespace b200moe

extern "C" int b200moe_route(const B200MoeRouteArgs* a, void* cuda_stream) {
  using namespace b200moe;
  if (!a) {
    set_error("null argument");
    return B200MOE_ERR_INVALID;
  }
  if (a->tokens < 0 || a->experts < 1 || a->experts > 256) {
    set_error("route: needs T >= 0, E in [1,256]");
    return B200MOE_ERR_INVALID;
  }
  if (!route_config_ok(a->config, a->experts, a->topk)) return B200MOE_ERR_INVALID;
  if (a->dtype != B200MOE_BF16 && a->dtype != B200MOE_FP16 && a->dtype != B200MOE_FP32) {
    set_error("route: unknown logits type %d", a->dtype);
    return B200MOE_ERR_INVALID;
  }
  if (static_cast<long long>(a->tokens) * a->topk >= (1LL << 31)) {
    set_error("route: T*K must stay below 2**31");
    return B200MOE_ERR_INVALID;
  }
  if (a->tokens == 0) return B200MOE_OK;
  if (a->pitch < a->experts && a->tokens > 1) {
    set_error("route: row pitch %lld is smaller than the %d experts", static_cast<long long>(a->pitch), a->experts);
    return B200MOE_ERR_INVALID;
  }
  if (!a->logits || !a->ids || !a->weights) {
    set_error("route: null buffer");
    return B200MOE_ERR_INVALID;
  }
  const uintptr_t element = a->dtype == B200MOE_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a->logits) % element || reinterpret_cast<uintptr_t>(a->ids) % (a->ids_are_int64 ? 8 : 4) ||
      reinterpret_cast<uintptr_t>(a->weights) % 4 || reinterpret_cast<uintptr_t>(a->bias) % 4) {
    set_error("route: misaligned buffer");
    return B200MOE_ERR_INVALID;
  }
  const route::Config cfg = route_config(a->config, a->experts, a->topk);
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  const cudaError_t e = a->dtype == B200MOE_FP32   ? launch_typed<float>(*a, cfg, s)
                        : a->dtype == B200MOE_BF16 ? launch_typed<__nv_bfloat16>(*a, cfg, s)
                                                   : launch_typed<__half>(*a, cfg, s);
  if (e != cudaSuccess) {
    set_error("route launch: %s", cudaGetErrorString(e));
    return B200MOE_ERR_CUDA;
  }
  return B200MOE_OK;
}
