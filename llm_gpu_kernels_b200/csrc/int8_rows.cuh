// Rows to 8-bit integers, one scale per row:
//   top = max |x_k|,  q_k = rint(127 x_k / top)  (ties to even),  scale = top / 127
// A row of zeros gives zeros and scale 0; a row that holds an infinity or a NaN gives zeros and scale NaN, so every
// product of it is NaN. q is that of exact arithmetic on the values read: x * (127 / top) in FP32 is off by at most
// 2^-16 (two roundings of values up to 127), so only a quotient that close to a half may round the wrong way, and
// those few are divided again in FP64 (where a 16-bit or 24-bit x over top cannot come closer to a half without being
// one than 2^-33).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace b200moe {
namespace rows8 {

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

// The factors of a row whose largest magnitude has the bits `bits`.
struct RowScale {
  float top, up, inverse, scale;
  bool zero;   // all of q is 0: a row of zeros, or one that is not finite
};
__device__ __forceinline__ RowScale row_scale_of(uint32_t bits) {
  RowScale r;
  const bool finite = bits < 0x7f800000u;
  r.top = __uint_as_float(bits);
  r.scale = finite ? r.top / 127.0f : __uint_as_float(0x7fffffffu);
  r.up = r.top < 1e-30f ? 0x1p100f : 1.0f;
  r.top *= r.up;
  r.zero = !finite || bits == 0;
  r.inverse = r.zero ? 0.0f : 127.0f / r.top;
  return r;
}
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], const RowScale& r) {
  return r.zero ? make_uint2(0u, 0u) : quantize8(v, r.inverse, r.top, r.up);
}

}  // namespace rows8
}  // namespace b200moe
