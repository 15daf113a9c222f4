// Rows to 8-bit integers in memory (the formula and its rounding: int8_rows.cuh).
// Bound by memory: it reads a row once (up to 32 values per thread stay in registers between the maximum and the
// rounding) and writes a byte per value; at a serving batch by launch latency.
#include "int8.h"
#include "int8_rows.cuh"
#include "pdl.cuh"

namespace b200moe {
namespace {

using namespace rows8;

constexpr int kThreads = 256;
constexpr int kCached = 4;   // pieces of 8 values a thread keeps

// L threads per row (a power of two, 32 .. 256).
template <typename T, int L, bool kVec>
__global__ void __launch_bounds__(kThreads)
quantize_rows_kernel(const T* __restrict__ x, long long pitch, int8_t* __restrict__ q, float* __restrict__ scale,
                     int rows, int K, int q_pitch) {
  pdl_launch_dependents();
  pdl_wait();   // x may be written by the kernel before; q may still be read by it
  const int t = threadIdx.x & (L - 1);
  const int row = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const bool live = row < rows;
  const T* src = x + static_cast<size_t>(live ? row : 0) * pitch;
  float v[kCached][8];
  uint32_t bits = 0;
#pragma unroll
  for (int c = 0; c < kCached; ++c) {
    load8<T, kVec>(src, (c * L + t) * 8, K, v[c]);
    bits = top_bits(v[c], bits);
  }
  for (int k = (kCached * L + t) * 8; k < K; k += L * 8) {
    float u[8];
    load8<T, kVec>(src, k, K, u);
    bits = top_bits(u, bits);
  }
  bits = __reduce_max_sync(0xffffffffu, bits);
  if (L > 32) {
    __shared__ uint32_t part[kThreads / 32];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = bits;
    __syncthreads();
    const int first = (threadIdx.x / L) * (L / 32);
#pragma unroll
    for (int w = 0; w < L / 32; ++w) bits = max(bits, part[first + w]);
  }
  if (!live) return;
  const RowScale r = row_scale_of(bits);
  if (t == 0) scale[row] = r.scale;
  int8_t* dst = q + static_cast<size_t>(row) * q_pitch;
#pragma unroll
  for (int c = 0; c < kCached; ++c) {
    const int k = (c * L + t) * 8;
    if (k < q_pitch) *reinterpret_cast<uint2*>(dst + k) = quantize8(v[c], r);
  }
  for (int k = (kCached * L + t) * 8; k < q_pitch; k += L * 8) {
    float u[8];
    load8<T, kVec>(src, k, K, u);
    *reinterpret_cast<uint2*>(dst + k) = quantize8(u, r);
  }
}

template <typename T, int L>
cudaError_t launch_rows(const QuantizeRows& a, cudaStream_t s) {
  const T* x = static_cast<const T*>(a.x);
  const bool vec = a.k % 8 == 0 && (a.pitch * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const int per_block = kThreads / L;
  const dim3 grid((a.rows + per_block - 1) / per_block);
  const int q_pitch = int8_pitch(a.k);
  return vec ? launch_pdl(quantize_rows_kernel<T, L, true>, grid, dim3(kThreads), 0, s, x, a.pitch, a.q, a.scale, a.rows,
                          a.k, q_pitch)
             : launch_pdl(quantize_rows_kernel<T, L, false>, grid, dim3(kThreads), 0, s, x, a.pitch, a.q, a.scale, a.rows,
                          a.k, q_pitch);
}

// As few threads per row as keep the row in registers.
template <typename T>
cudaError_t launch_typed(const QuantizeRows& a, cudaStream_t s) {
  if (a.k <= 32 * 8 * kCached) return launch_rows<T, 32>(a, s);
  if (a.k <= 64 * 8 * kCached) return launch_rows<T, 64>(a, s);
  if (a.k <= 128 * 8 * kCached) return launch_rows<T, 128>(a, s);
  return launch_rows<T, 256>(a, s);
}

}  // namespace

cudaError_t launch_quantize_rows(const QuantizeRows& a, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  if (a.dtype == B200MOE_BF16) return launch_typed<__nv_bfloat16>(a, s);
  if (a.dtype == B200MOE_FP16) return launch_typed<__half>(a, s);
  return launch_typed<float>(a, s);
}

}  // namespace b200moe
