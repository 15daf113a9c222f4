// Rows to 8-bit integers, one scale per row:
//   top = max |x_k|,  q_k = rint(127 x_k / top)  (ties to even),  scale = top / 127
// A row of zeros gives zeros and scale 0; a row that holds an infinity or a NaN gives zeros and scale NaN, so every
// product of it is NaN. q is that of exact arithmetic on the values read (quantize8).
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

// sum * row scale * channel scale. The product of the two scales comes first, one rounding (and in a tile one
// multiplication) less per value. Where it leaves FP32's normal range, as with rows of 1e-35 and channels of 1e-6, the
// result may still be in it; then the larger scale goes first. If the product is too small the larger is below 2^23
// (nothing is below 2^-149) and |sum| below 2^31, so nothing overflows and only the last step may be subnormal; if it is
// too large the result is an infinity, or 0 for a sum of 0. Selects and no branch: a second path costs short kernels more,
// which fetch their instructions cold.
__device__ __forceinline__ bool in_range(float scale) { return fabsf(scale) >= 0x1p-126f && fabsf(scale) < INFINITY; }
__device__ __forceinline__ float scaled(int sum, float row, float channel) {
  const float scale = row * channel;
  const bool near = in_range(scale), channel_first = fabsf(channel) > row;
  return static_cast<float>(sum) * (near ? scale : channel_first ? channel : row) * (near ? 1.0f : channel_first ? row : channel);
}

// The factors of a row whose largest magnitude has the bits `bits`.
struct RowScale {
  float up;                          // a power of two that keeps the row clear of overflow and of subnormals
  float top, reciprocal, inverse;    // the largest magnitude times up, 1 / top, 127 / top
  float scale;
  bool zero;   // all of q is 0: a row of zeros, or one that is not finite
};
__device__ __forceinline__ RowScale row_scale_of(uint32_t bits) {
  RowScale r;
  const bool finite = bits < 0x7f800000u;
  r.top = __uint_as_float(bits);
  r.scale = finite ? r.top / 127.0f : __uint_as_float(0x7fffffffu);
  r.up = r.top < 1e-30f ? 0x1p100f : r.top > 1e30f ? 0x1p-100f : 1.0f;
  r.top *= r.up;
  r.zero = !finite || bits == 0;
  r.inverse = r.zero ? 0.0f : 127.0f / r.top;
  r.reciprocal = r.zero ? 0.0f : 1.0f / r.top;
  return r;
}
__device__ __forceinline__ uint2 pack8(const uint32_t (&b)[8]) {   // the low bytes
  return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// Eight values to eight bytes, six or seven instructions each. Adding 1.5 * 2^23 rounds to an integer, ties to even, and
// leaves it in the low bits.
// kHalf (16-bit values): 127 x is exact in FP32, and one correction with its exact remainder gives the quotient with an
// error below 2^-16; a quotient that is a half exactly is representable and comes out exact, any other is at least
// 2^-12 away from a half (denominators below 2^11): no quotient rounds the wrong way.
// FP32 values: the quotient is off by up to 2^-16; where one of the eight is that close to a half, they are divided in FP64.
template <bool kHalf>
__device__ __forceinline__ uint2 quantize8(const float (&v)[8], const RowScale& r) {
  if (r.zero) return make_uint2(0u, 0u);
  constexpr float kRound = 12582912.0f;
  uint32_t b[8];
  if (kHalf) {
    const float factor = 127.0f * r.up;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float p = v[j] * factor;
      const float t = p * r.reciprocal;
      b[j] = __float_as_uint(__fadd_rn(fmaf(fmaf(-t, r.top, p), r.reciprocal, t), kRound));
    }
    return pack8(b);
  }
  float far = 0.0f;   // the largest distance from an integer
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = v[j] * r.inverse;
    const float q = __fadd_rn(t, kRound);
    far = fmaxf(far, fabsf(__fsub_rn(t, __fsub_rn(q, kRound))));
    b[j] = __float_as_uint(q);
  }
  if (far > 0.49998f || r.up != 1.0f) {   // one test for all eight: a branch per value costs more than the rounding
#pragma unroll
    for (int j = 0; j < 8; ++j)
      b[j] = static_cast<uint32_t>(
          static_cast<int>(rint(127.0 * static_cast<double>(v[j]) * r.up / static_cast<double>(r.top))));
  }
  return pack8(b);
}

}  // namespace rows8
}  // namespace b200moe
