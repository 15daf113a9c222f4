// Rows to 8-bit integers in memory (the formula and its rounding: int8_rows.cuh).
// Bound by memory: it reads a row once (up to 32 values per thread stay in registers between the maximum and the
// rounding) and writes a byte per value; at a serving batch by launch latency. Six or seven instructions per value
// keep it from the copy rate where rows are many: 1024 x 2048 BF16 5.5 us, 8192 x 4096 BF16 23 us (4.4 TB/s, issue slots
// 69 %), 8192 x 768 FP32 10.4 us (3.0 TB/s).
#include "int8.h"
#include "int8_rows.cuh"
#include "pdl.cuh"

namespace b200moe {
namespace {

using namespace rows8;

constexpr int kThreads = 256;
constexpr int kCached = 4;   // pieces of 8 values a thread keeps

// L threads per row (a power of two, 32 .. 256). kScatter: row r goes to the rows mapping[r * copies ..] of q and scale
// instead of row r (the grouped rows of the token's routes; negative: none).
template <typename T, int L, bool kVec, bool kScatter>
__global__ void __launch_bounds__(kThreads)
quantize_rows_kernel(const T* __restrict__ x, long long pitch, int8_t* __restrict__ q, float* __restrict__ scale,
                     int rows, int K, int q_pitch, const int* __restrict__ mapping, int copies) {
  pdl_wait();   // x may be written by the kernel before; q may still be read by it
  pdl_launch_dependents();   // not earlier: a dependent relies on everything before this kernel being complete
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
  if (!kScatter && t == 0) scale[row] = r.scale;
  if (kScatter)
    for (int c = t; c < copies; c += L) {
      const int to = mapping[static_cast<size_t>(row) * copies + c];
      if (to >= 0) scale[to] = r.scale;
    }
  auto store = [&](int k, uint2 v8) {
    if (!kScatter) {
      *reinterpret_cast<uint2*>(q + static_cast<size_t>(row) * q_pitch + k) = v8;
    } else {
      for (int c = 0; c < copies; ++c) {
        const int to = mapping[static_cast<size_t>(row) * copies + c];
        if (to >= 0) *reinterpret_cast<uint2*>(q + static_cast<size_t>(to) * q_pitch + k) = v8;
      }
    }
  };
#pragma unroll
  for (int c = 0; c < kCached; ++c) {
    const int k = (c * L + t) * 8;
    if (k < q_pitch) store(k, quantize8<sizeof(T) == 2>(v[c], r));
  }
  for (int k = (kCached * L + t) * 8; k < q_pitch; k += L * 8) {
    float u[8];
    load8<T, kVec>(src, k, K, u);
    store(k, quantize8<sizeof(T) == 2>(u, r));
  }
}

template <typename T, int L>
cudaError_t launch_rows(const QuantizeRows& a, cudaStream_t s) {
  const T* x = static_cast<const T*>(a.x);
  const bool vec = a.k % 8 == 0 && (a.pitch * sizeof(T)) % 16 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  const int per_block = kThreads / L;
  const dim3 grid((a.rows + per_block - 1) / per_block);
  const int q_pitch = int8_pitch(a.k);
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, grid, dim3(kThreads), 0, s, x, a.pitch, a.q, a.scale, a.rows, a.k, q_pitch, a.mapping, a.copies);
  };
  if constexpr (sizeof(T) == 2)
    if (a.mapping) return vec ? go(quantize_rows_kernel<T, L, true, true>) : go(quantize_rows_kernel<T, L, false, true>);
  return vec ? go(quantize_rows_kernel<T, L, true, false>) : go(quantize_rows_kernel<T, L, false, false>);
}

// As few threads per row as keep the row in registers; with few rows, as many as have a piece to do (latency).
template <typename T>
cudaError_t launch_typed(const QuantizeRows& a, cudaStream_t s) {
  const int per = a.rows <= 256 ? 8 : 8 * kCached;
  if (a.k <= 32 * per) return launch_rows<T, 32>(a, s);
  if (a.k <= 64 * per) return launch_rows<T, 64>(a, s);
  if (a.k <= 128 * per) return launch_rows<T, 128>(a, s);
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
