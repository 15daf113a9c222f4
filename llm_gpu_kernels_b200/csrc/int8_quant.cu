// Rows to 8-bit integers, one scale per row:
//   top = max |x_k|,  q_k = rint(127 x_k / top)  (ties to even),  scale = top / 127
// A row of zeros gives zeros and scale 0; a row that holds an infinity or a NaN gives zeros and scale NaN, so every
// product of it is NaN. q is that of exact arithmetic on the values read: x * (127 / top) in FP32 is off by at most
// 2^-16 (two roundings of values up to 127), so only a quotient that close to a half may round the wrong way, and
// those few are divided again in FP64 (where a 16-bit or 24-bit x over top cannot come closer to a half without being
// one than 2^-33).
// Bound by memory: it reads a row once (up to 32 values per thread stay in registers between the maximum and the
// rounding) and writes a byte per value; at a serving batch by launch latency.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "int8.h"
#include "pdl.cuh"

namespace b200moe {
namespace {

constexpr int kThreads = 256;
constexpr int kCached = 4;   // pieces of 8 values a thread keeps

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

// Values k .. k+7 of a row, zero past its end.
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T* __restrict__ row, int k, int K, float (&v)[8]) {
  if (kVec) {
    union { T t[8]; uint4 q[sizeof(T) / 2]; } raw;
    if (k < K) {   // K is a multiple of 8 here
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) raw.q[i] = *(reinterpret_cast<const uint4*>(row + k) + i);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_float(raw.t[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? to_float(row[k + j]) : 0.0f;
  }
}

__device__ __forceinline__ uint32_t top_bits(const float (&v)[8], uint32_t top) {
#pragma unroll
  for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);   // NaN > Inf > finite
  return top;
}

// up: a power of two that lifts the row out of the subnormal range.
__device__ __forceinline__ int round_to_int8(float x, float inverse, float top, float up) {
  const float t = x * up * inverse, r = rintf(t);
  if (fabsf(t - r) > 0.4999f) return static_cast<int>(rint(127.0 * static_cast<double>(x) * up / static_cast<double>(top)));
  return static_cast<int>(r);
}

__device__ __forceinline__ uint2 quantize8(const float (&v)[8], float inverse, float top, float up) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    w[j >> 2] |= (static_cast<uint32_t>(round_to_int8(v[j], inverse, top, up)) & 0xffu) << (8 * (j & 3));
  return make_uint2(w[0], w[1]);
}

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
  const bool finite = bits < 0x7f800000u;
  float top = __uint_as_float(bits);
  if (t == 0) scale[row] = finite ? top / 127.0f : __uint_as_float(0x7fffffffu);
  const float up = top < 1e-30f ? 0x1p100f : 1.0f;
  top *= up;
  const bool zero = !finite || bits == 0;
  const float inverse = zero ? 0.0f : 127.0f / top;
  int8_t* dst = q + static_cast<size_t>(row) * q_pitch;
#pragma unroll
  for (int c = 0; c < kCached; ++c) {
    const int k = (c * L + t) * 8;
    if (k < q_pitch) *reinterpret_cast<uint2*>(dst + k) = zero ? make_uint2(0u, 0u) : quantize8(v[c], inverse, top, up);
  }
  for (int k = (kCached * L + t) * 8; k < q_pitch; k += L * 8) {
    float u[8];
    load8<T, kVec>(src, k, K, u);
    *reinterpret_cast<uint2*>(dst + k) = zero ? make_uint2(0u, 0u) : quantize8(u, inverse, top, up);
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
