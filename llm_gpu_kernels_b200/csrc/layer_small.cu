// The two products of an INT8 layer for a few routes (a decode step), without tensor cores. Every block works on one
// route: it quantises the route's row (of x, or of the activated rows) into its shared memory, then its warps take
// channels of the route's expert in turn, as the dense product for one token does (linear_small.cu): 32 lanes read 512
// bytes of two weight rows at a time - the gate and the up row of a channel, or two neighbouring channels of the down
// product - with four-way integer dot products and one warp reduction per row. Sums are exact, so the results are those
// of the tensor-core kernels to the bit.
// Bound by the stream of weights, one pass per route (38 MB for 8 routes of 2048 x 768 experts: 5.8 us), and by the
// launches: two kernels here against four (two quantisations, two products). Two blocks per SM: with three or four the
// registers do not hold the weights in flight (1 token x 8 experts 20.8 and 24.6 us). __expf as in grouped_gemm_i8.cu.
#include "int8.h"
#include "int8_rows.cuh"
#include "pdl.cuh"

namespace b200moe {
namespace {

using namespace rows8;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPieces = 4;              // 16-byte pieces of each weight row a lane has in flight
constexpr int kRound = 512 * kPieces;

// kGateUp: T = BF16 rows of x, one per token; else T = float, activated rows in grouped order.
template <bool kGateUp, typename T, typename IdT, bool kVec>
__global__ void __launch_bounds__(kThreads, 2)
layer_small_kernel(const LayerSmall a) {
  extern __shared__ __align__(16) unsigned char smem[];   // the row as int8, zero past its end
  __shared__ uint32_t part[kWarps];
  pdl_launch_dependents();
  pdl_wait();
  const int route = blockIdx.y;
  const int at = a.mapping[route];        // the route's grouped row
  const long long expert = static_cast<const IdT*>(a.ids)[route];
  if (at < 0 || expert < 0 || expert >= a.experts) return;
  const int row = kGateUp ? route / a.topk : at;
  const T* x = static_cast<const T*>(a.x) + static_cast<size_t>(row) * a.k;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pitch = int8_pitch(a.k), smem_pitch = (a.k + 511) / 512 * 512;
  const int8_t* w = a.weight + static_cast<size_t>(expert) * a.w_rows * pitch;
  const float* w_scale = a.w_scale + static_cast<size_t>(expert) * a.w_rows;
  const int stride = kGateUp ? 1 : 2;     // channels per step of a warp
  const int second = kGateUp ? a.n_out : 1;
  const int step = static_cast<int>(gridDim.x) * kWarps * stride;
  int n = (blockIdx.x * kWarps + warp) * stride;
  uint4 ahead[2][kPieces];
  auto fetch = [&](int n, int k0) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int k = k0 + i * 512 + lane * 16;
        const bool there = k < pitch && n < a.n_out && (kGateUp || n + c < a.n_out);
        ahead[c][i] = there ? __ldg(reinterpret_cast<const uint4*>(w + static_cast<size_t>(n + c * second) * pitch + k))
                            : make_uint4(0u, 0u, 0u, 0u);
      }
  };
  fetch(n, 0);   // on their way while the row is quantised
  uint32_t bits = 0;
  for (int k = threadIdx.x * 8; k < a.k; k += kThreads * 8) {
    float v[8];
    load8<T, kVec>(x, k, a.k, v);
    bits = top_bits(v, bits);
  }
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (lane == 0) part[warp] = bits;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) bits = max(bits, part[i]);
  const RowScale scale = row_scale_of(bits);
  const bool keep = blockIdx.x == 0;   // one block per route leaves its row in memory too, in grouped order
  if (keep && threadIdx.x == 0) a.q_scale[at] = scale.scale;
  for (int k = threadIdx.x * 8; k < smem_pitch; k += kThreads * 8) {
    float v[8] = {};
    load8<T, kVec>(x, k, a.k, v);
    const uint2 q = quantize8<sizeof(T) == 2>(v, scale);
    *reinterpret_cast<uint2*>(smem + k) = q;
    if (keep && k < pitch) *reinterpret_cast<uint2*>(a.q + static_cast<size_t>(at) * pitch + k) = q;
  }
  __syncthreads();
  for (; n < a.n_out; n += step) {
    int acc[2] = {0, 0};
    for (int k0 = 0; k0 < pitch; k0 += kRound) {
      uint4 now[2][kPieces];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < kPieces; ++i) now[c][i] = ahead[c][i];
      if (k0 + kRound < pitch) fetch(n, k0 + kRound);
      else fetch(n + step, 0);
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int k = k0 + i * 512 + lane * 16;
        const uint4 q = k < smem_pitch ? *reinterpret_cast<const uint4*>(smem + k) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          acc[c] = __dp4a(static_cast<int>(now[c][i].x), static_cast<int>(q.x), acc[c]);
          acc[c] = __dp4a(static_cast<int>(now[c][i].y), static_cast<int>(q.y), acc[c]);
          acc[c] = __dp4a(static_cast<int>(now[c][i].z), static_cast<int>(q.z), acc[c]);
          acc[c] = __dp4a(static_cast<int>(now[c][i].w), static_cast<int>(q.w), acc[c]);
        }
      }
    }
    const int s0 = __reduce_add_sync(0xffffffffu, acc[0]), s1 = __reduce_add_sync(0xffffffffu, acc[1]);
    const size_t out = static_cast<size_t>(at) * a.n_out + n;
    if (kGateUp) {
      if (lane == 0) {
        const float gate = scaled(s0, scale.scale, w_scale[n]);
        const float up = scaled(s1, scale.scale, w_scale[n + second]);
        a.y[out] = (gate / (1.0f + __expf(-gate))) * up;
      }
    } else if (lane < 2 && n + lane < a.n_out) {
      a.y[out + lane] = scaled(lane ? s1 : s0, scale.scale, w_scale[n + lane]);
    }
  }
}

template <bool kGateUp, typename T, typename IdT>
cudaError_t launch(const LayerSmall& a, int sms, cudaStream_t s) {
  const bool vec = a.k % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
  const int per_block = kWarps * (kGateUp ? 1 : 2);
  int blocks = (a.n_out + per_block - 1) / per_block;
  const int most = (sms * 2 + a.routes - 1) / a.routes;   // two blocks per SM are resident
  if (blocks > most) blocks = most;
  const dim3 grid(blocks, a.routes);
  const size_t smem = (a.k + 511) / 512 * 512;
  return vec ? launch_pdl(layer_small_kernel<kGateUp, T, IdT, true>, grid, dim3(kThreads), smem, s, a)
             : launch_pdl(layer_small_kernel<kGateUp, T, IdT, false>, grid, dim3(kThreads), smem, s, a);
}

}  // namespace

// One token of at most eight routes, two of at most two each: an expert's weights cross once per route here, once per
// tile of rows there. A forward without / with tensor cores: 20.5 / 24.6 us for 1 token x 8 of 128 experts 2048 x 768,
// 36.6 / 33.4 us for 2; 72 / 76, 107 / 105, 234 / 154 us for 1, 2, 3 tokens x 2 of 8 experts 4096 x 14336.
bool layer_small_serves(int tokens, int topk, int hidden, int intermediate) {
  const int widest = hidden > intermediate ? hidden : intermediate;
  return ((tokens == 1 && topk <= 8) || (tokens == 2 && topk <= 2)) && widest <= 46 * 1024;
}

cudaError_t launch_layer_small(const LayerSmall& a, bool gate_up, int sms, cudaStream_t s) {
  if (gate_up)
    return a.ids_are_int64 ? launch<true, __nv_bfloat16, long long>(a, sms, s) : launch<true, __nv_bfloat16, int>(a, sms, s);
  return a.ids_are_int64 ? launch<false, float, long long>(a, sms, s) : launch<false, float, int>(a, sms, s);
}

}  // namespace b200moe
