// The dense 8-bit product for one or two tokens (a decode step): one launch, no tensor cores.
// Every block quantises the rows of x into its shared memory (int8_rows.cuh; a few KB out of L2, hidden behind the first
// weight loads, which are issued before), then its warps take output channels in turn: 32 lanes read 512 bytes of a
// weight row at a time, 16 bytes each, multiply with four-way integer dot products and add up with one warp reduction.
// Bound by the stream of weights (N * K bytes, read once) and for a small weight by
// launch and load latency: 3.0 us for 1 x 2048 x 1536, 6.4 us for 4096 x 4096, 12.4 us for 4096 x 14336 (4.75 TB/s).
#include "int8.h"
#include "int8_rows.cuh"
#include "pdl.cuh"

namespace b200moe {
namespace {

using namespace rows8;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPieces = 4;                 // 16-byte pieces of a weight row a lane has in flight
constexpr int kRound = 512 * kPieces;      // bytes of a weight row a warp has in flight

__device__ __forceinline__ void store_out(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_out(__half* p, float v) { *p = __float2half_rn(v); }

// kRows: tokens (rounded up); kCh: output channels a warp works on at the same time.
template <typename T, int kRows, int kCh, bool kVec>
__global__ void __launch_bounds__(kThreads)
linear_small_kernel(const T* __restrict__ x, long long x_pitch, const int8_t* __restrict__ w,
                    const float* __restrict__ w_scale, T* __restrict__ y, int8_t* __restrict__ x_q,
                    float* __restrict__ x_scale, int tokens, int K, int N, int pitch, int smem_pitch) {
  extern __shared__ __align__(16) unsigned char smem[];   // [kRows][smem_pitch] int8, zero past K
  __shared__ uint32_t part[kRows][kWarps];
  __shared__ float row_scale[kRows];
  pdl_launch_dependents();
  pdl_wait();   // x may be written by the kernel before; y may still be read by it
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int step = static_cast<int>(gridDim.x) * kWarps * kCh;
  int n0 = (blockIdx.x * kWarps + warp) * kCh;
  uint4 ahead[kCh][kPieces];               // the first pieces of the channels to come
  auto fetch = [&](int n, int k0) {
#pragma unroll
    for (int c = 0; c < kCh; ++c)
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int k = k0 + i * 512 + lane * 16;
        ahead[c][i] = n + c < N && k < pitch ? __ldg(reinterpret_cast<const uint4*>(w + static_cast<size_t>(n + c) * pitch + k))
                                             : make_uint4(0u, 0u, 0u, 0u);
      }
  };
  fetch(n0, 0);
  uint32_t bits[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    bits[r] = 0;
    for (int k = threadIdx.x * 8; k < K && r < tokens; k += kThreads * 8) {
      float v[8];
      load8<T, kVec>(x + r * x_pitch, k, K, v);
      bits[r] = top_bits(v, bits[r]);
    }
    bits[r] = __reduce_max_sync(0xffffffffu, bits[r]);
    if (lane == 0) part[r][warp] = bits[r];
  }
  __syncthreads();
  const bool keep = blockIdx.x == 0;       // one block leaves the rows in memory too
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
#pragma unroll
    for (int i = 0; i < kWarps; ++i) bits[r] = max(bits[r], part[r][i]);
    const RowScale s = row_scale_of(bits[r]);
    if (threadIdx.x == r) row_scale[r] = s.scale;
    if (keep && threadIdx.x == r && r < tokens) x_scale[r] = s.scale;
    for (int k = threadIdx.x * 8; k < smem_pitch; k += kThreads * 8) {
      float v[8] = {};
      if (r < tokens) load8<T, kVec>(x + r * x_pitch, k, K, v);
      const uint2 q = quantize8<true>(v, s);
      *reinterpret_cast<uint2*>(smem + r * smem_pitch + k) = q;
      if (keep && k < pitch && r < tokens) *reinterpret_cast<uint2*>(x_q + static_cast<size_t>(r) * pitch + k) = q;
    }
  }
  __syncthreads();
  for (; n0 < N; n0 += step) {
    int acc[kCh][kRows] = {};
    for (int k0 = 0; k0 < pitch; k0 += kRound) {
      uint4 now[kCh][kPieces];
#pragma unroll
      for (int c = 0; c < kCh; ++c)
#pragma unroll
        for (int i = 0; i < kPieces; ++i) now[c][i] = ahead[c][i];
      if (k0 + kRound < pitch) fetch(n0, k0 + kRound);
      else fetch(n0 + step, 0);            // zeros past the last channel
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int k = k0 + i * 512 + lane * 16;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const uint4 q = k < smem_pitch ? *reinterpret_cast<const uint4*>(smem + r * smem_pitch + k) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
          for (int c = 0; c < kCh; ++c) {
            int a = acc[c][r];
            a = __dp4a(static_cast<int>(now[c][i].x), static_cast<int>(q.x), a);
            a = __dp4a(static_cast<int>(now[c][i].y), static_cast<int>(q.y), a);
            a = __dp4a(static_cast<int>(now[c][i].z), static_cast<int>(q.z), a);
            acc[c][r] = __dp4a(static_cast<int>(now[c][i].w), static_cast<int>(q.w), a);
          }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kCh; ++c)
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int sum = __reduce_add_sync(0xffffffffu, acc[c][r]);
        if (lane == c * kRows + r && n0 + c < N && r < tokens)
          store_out(y + static_cast<size_t>(r) * N + n0 + c, scaled(sum, row_scale[r], w_scale[n0 + c]));
      }
  }
}

int smem_pitch_of(int k) { return (k + 511) / 512 * 512; }

template <typename T, int kRows, int kCh>
cudaError_t launch(const LinearSmall& a, cudaStream_t s) {
  const T* x = static_cast<const T*>(a.x);
  const bool vec = a.k % 8 == 0 && (a.x_pitch * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const int blocks = (a.n + kWarps * kCh - 1) / (kWarps * kCh), most = a.sms * 4;
  const dim3 grid(blocks < most ? blocks : most);
  const int pitch = smem_pitch_of(a.k);
  const size_t smem = static_cast<size_t>(kRows) * pitch;
  return vec ? launch_pdl(linear_small_kernel<T, kRows, kCh, true>, grid, dim3(kThreads), smem, s, x, a.x_pitch, a.weight,
                          a.w_scale, static_cast<T*>(a.y), a.q, a.q_scale, a.tokens, a.k, a.n, int8_pitch(a.k), pitch)
             : launch_pdl(linear_small_kernel<T, kRows, kCh, false>, grid, dim3(kThreads), smem, s, x, a.x_pitch, a.weight,
                          a.w_scale, static_cast<T*>(a.y), a.q, a.q_scale, a.tokens, a.k, a.n, int8_pitch(a.k), pitch);
}

template <typename T>
cudaError_t launch_typed(const LinearSmall& a, cudaStream_t s) {
  return a.tokens == 1 ? launch<T, 1, 1>(a, s) : launch<T, 2, 2>(a, s);
}

}  // namespace

// One token, or two with a weight of at most 32 MB: the second token costs as much again in dot products and shared
// memory reads, the tensor cores nothing (two tokens: 4.4 against 6.2 us at 2048 x 1536, 8.3 against 9.6 at 4096 x 4096,
// 19.5 against 15.8 at 4096 x 14336; four tokens would take 7.1, 12.5 and 27 us). Their quantised rows have to fit the
// shared memory a block has without opting in.
bool linear_small_serves(int tokens, int k, int n) {
  return (tokens == 1 || (tokens == 2 && static_cast<long long>(n) * k <= 32ll << 20)) &&
         static_cast<long long>(tokens) * smem_pitch_of(k) <= 46 * 1024;
}

cudaError_t launch_linear_small(const LinearSmall& a, cudaStream_t s) {
  return a.dtype == B200MOE_BF16 ? launch_typed<__nv_bfloat16>(a, s) : launch_typed<__half>(a, s);
}

}  // namespace b200moe
