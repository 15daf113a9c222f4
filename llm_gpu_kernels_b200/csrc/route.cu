// Routing on given logits: [T, E] in BF16, FP16 or FP32 (rows may be strided) to ids and weights [T, K]. The formula is
// in route_row.cuh; a row is held in registers by 32, 16, 8 or 4 lanes, up to 8 experts each, and read once.
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

// kVec: a lane's P logits are one aligned piece (E a multiple of P, row pitch and base aligned to P elements).
template <typename T, typename IdT, int P, int L, bool kVec>
__global__ void __launch_bounds__(kThreads)
route_kernel(const T* __restrict__ logits, long long pitch, const float* __restrict__ bias, IdT* __restrict__ ids,
             float* __restrict__ weights, int tokens, const __grid_constant__ route::Config cfg) {
  pdl_launch_dependents();
  pdl_wait();   // the logits may come from the kernel just before; ids / weights may still be read by it
  const int lane = threadIdx.x & (L - 1);
  const long long row = static_cast<long long>(blockIdx.x) * (kThreads / L) + threadIdx.x / L;
  if (row >= tokens) return;
  const unsigned mask = L == 32 ? 0xffffffffu : ((1u << L) - 1u) << ((threadIdx.x & 31) & ~(L - 1));
  const T* src = logits + row * pitch + lane * P;
  float l[P];
  if (kVec) {
    union { T v[P]; uint32_t w[(P * sizeof(T) + 3) / 4]; } raw;
    if (lane * P < cfg.E) {
      constexpr int kBytes = P * sizeof(T);
      if constexpr (kBytes % 16 == 0) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) {
          const uint4 q = __ldg(reinterpret_cast<const uint4*>(src) + i);
          raw.w[4 * i] = q.x; raw.w[4 * i + 1] = q.y; raw.w[4 * i + 2] = q.z; raw.w[4 * i + 3] = q.w;
        }
      } else if constexpr (kBytes == 8) {
        const uint2 q = __ldg(reinterpret_cast<const uint2*>(src));
        raw.w[0] = q.x; raw.w[1] = q.y;
      } else {
#pragma unroll
        for (int i = 0; i < P; ++i) raw.v[i] = src[i];
      }
#pragma unroll
      for (int j = 0; j < P; ++j) l[j] = to_float(raw.v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) l[j] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int j = 0; j < P; ++j) l[j] = lane * P + j < cfg.E ? to_float(src[j]) : -INFINITY;
  }
  route::route_row<P, L, IdT>(cfg, l, bias, lane, mask, ids + row * cfg.K, weights + row * cfg.K);
}

template <typename T, typename IdT, int P, int L>
cudaError_t launch(const B200MoeRouteArgs& a, const route::Config& cfg, cudaStream_t s) {
  const T* logits = static_cast<const T*>(a.logits);
  const bool vec = cfg.E % P == 0 && a.pitch % P == 0 && reinterpret_cast<uintptr_t>(logits) % 16 == 0 &&
                   (a.pitch * sizeof(T)) % (P * sizeof(T) < 16 ? P * sizeof(T) : 16) == 0;
  const int rows = kThreads / L;
  const dim3 grid(static_cast<unsigned>((static_cast<long long>(a.tokens) + rows - 1) / rows));
  auto* ids = static_cast<IdT*>(a.ids);
  auto* w = static_cast<float*>(a.weights);
  auto* bias = static_cast<const float*>(a.bias);
  return vec ? launch_pdl(route_kernel<T, IdT, P, L, true>, grid, dim3(kThreads), 0, s, logits,
                          static_cast<long long>(a.pitch), bias, ids, w, a.tokens, cfg)
             : launch_pdl(route_kernel<T, IdT, P, L, false>, grid, dim3(kThreads), 0, s, logits,
                          static_cast<long long>(a.pitch), bias, ids, w, a.tokens, cfg);
}

// Lanes per row: eight experts per lane where that leaves at least four lanes, so that small expert counts share a
// warp among several rows. Groups need the whole warp (one lane per group).
template <typename T, typename IdT>
cudaError_t launch_shape(const B200MoeRouteArgs& a, const route::Config& cfg, cudaStream_t s) {
  if (cfg.groups > 1 || cfg.E > 128) {
    if (cfg.E <= 32) return launch<T, IdT, 1, 32>(a, cfg, s);
    if (cfg.E <= 64) return launch<T, IdT, 2, 32>(a, cfg, s);
    if (cfg.E <= 128) return launch<T, IdT, 4, 32>(a, cfg, s);
    return launch<T, IdT, 8, 32>(a, cfg, s);
  }
  if (cfg.E <= 32) return launch<T, IdT, 8, 4>(a, cfg, s);
  if (cfg.E <= 64) return launch<T, IdT, 8, 8>(a, cfg, s);
  return launch<T, IdT, 8, 16>(a, cfg, s);
}

template <typename T>
cudaError_t launch_typed(const B200MoeRouteArgs& a, const route::Config& cfg, cudaStream_t s) {
  return a.ids_are_int64 ? launch_shape<T, long long>(a, cfg, s) : launch_shape<T, int>(a, cfg, s);
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
