// Weighted combine back to token order:
//   out[t,:] = bf16( sum_{slot=0..K-1} float(down_output[mapping[t*K+slot],:]) * rw[t,slot] )
// (the rows are BF16, or FP32 in an INT8 plan)
// in fixed slot order, FP32, multiply and add kept as separate roundings -
// the semantics of the reference's _combine (moe.py:109-121, launched with
// enable_fp_fusion=False at moe.py:217). A gather-reduce, not a scatter with
// atomics, so the result does not depend on scheduling. Routes with
// mapping < 0 (invalid expert id) contribute nothing (moe.py:117).
// Optional residual: out = bf16(float(residual[t,:]) + float(bf16(sum))) - what the layer followed by the
// model's BF16 residual add gives, without writing and re-reading the layer output.
#include <cuda_bf16.h>
#include "plan.h"
#include "pdl.cuh"

namespace b200moe {
namespace {

constexpr int kThreads = 64;  // small blocks: T * H/512 of them even for a handful of tokens

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// The values of a 16-byte piece of a row.
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x);
  f[1] = __uint_as_float(v.y);
  f[2] = __uint_as_float(v.z);
  f[3] = __uint_as_float(v.w);
}

// kScalar: values per thread where rows are not aligned. In: type of the rows; aligned ones are read 16 bytes per thread
// and row.
template <typename In, bool kVec, int kScalar>
__global__ void __launch_bounds__(kThreads)
combine_kernel(const In* __restrict__ down_out, const int* __restrict__ mapping,
               const float* __restrict__ rw, __nv_bfloat16* __restrict__ out, const int* __restrict__ valid_routes,
               const __nv_bfloat16* __restrict__ residual, int H, int K) {
  pdl_launch_dependents();
  pdl_wait();  // down_output / mapping come from the kernels before
  const int token = blockIdx.x;
  if (valid_routes && token * K >= *valid_routes) return;  // padding rows of a fixed-capacity buffer
  __shared__ int s_pos[32];
  __shared__ float s_w[32];
  if (threadIdx.x < K) {
    s_pos[threadIdx.x] = mapping[static_cast<size_t>(token) * K + threadIdx.x];
    s_w[threadIdx.x] = rw[static_cast<size_t>(token) * K + threadIdx.x];
  }
  __syncthreads();
  if (kVec) {
    constexpr int N = 16 / sizeof(In);
    struct alignas(2 * N) Piece { uint32_t u[N / 2]; };   // N values in BF16
    const int h = (blockIdx.y * kThreads + threadIdx.x) * N;
    if (h >= H) return;
    float acc[N] = {};
    for (int s0 = 0; s0 < K; s0 += 8) {  // issue the (independent) row loads first, then add in slot order
      uint4 v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int slot = s0 + j;
        const int pos = slot < K ? s_pos[slot] : -1;
        v[j] = pos >= 0 ? *reinterpret_cast<const uint4*>(down_out + static_cast<size_t>(pos) * H + h)
                        : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int slot = s0 + j;
        if (slot >= K || s_pos[slot] < 0) continue;
        const float w = s_w[slot];
        float f[N];
        unpack(v[j], f);
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = __fadd_rn(acc[i], __fmul_rn(f[i], w));
      }
    }
    Piece o;
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(acc[2 * j], acc[2 * j + 1]);
      o.u[j] = *reinterpret_cast<const uint32_t*>(&v);
    }
    if (residual) {
      const Piece r = *reinterpret_cast<const Piece*>(residual + static_cast<size_t>(token) * H + h);
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(
            __fadd_rn(__uint_as_float(r.u[j] << 16), __uint_as_float(o.u[j] << 16)),
            __fadd_rn(__uint_as_float(r.u[j] & 0xffff0000u), __uint_as_float(o.u[j] & 0xffff0000u)));
        o.u[j] = *reinterpret_cast<const uint32_t*>(&v);
      }
    }
    *reinterpret_cast<Piece*>(out + static_cast<size_t>(token) * H + h) = o;
  } else {
    const int h0 = blockIdx.y * kThreads * kScalar + threadIdx.x;
    float acc[kScalar] = {};
    for (int slot = 0; slot < K; ++slot) {
      const int pos = s_pos[slot];
      if (pos < 0) continue;
      const In* row = down_out + static_cast<size_t>(pos) * H;
#pragma unroll
      for (int j = 0; j < kScalar; ++j) {
        const int h = h0 + j * kThreads;
        if (h < H) acc[j] = __fadd_rn(acc[j], __fmul_rn(to_float(row[h]), s_w[slot]));
      }
    }
#pragma unroll
    for (int j = 0; j < kScalar; ++j) {
      const int h = h0 + j * kThreads;
      if (h >= H) break;
      __nv_bfloat16 r = __float2bfloat16_rn(acc[j]);
      if (residual)
        r = __float2bfloat16_rn(__fadd_rn(__bfloat162float(residual[static_cast<size_t>(token) * H + h]), __bfloat162float(r)));
      out[static_cast<size_t>(token) * H + h] = r;
    }
  }
}

template <typename In>
void launch_typed(const B200MoePlan& p, cudaStream_t s) {
  const auto& sh = p.shape;
  auto* d = static_cast<const In*>(p.buf.down_output);
  auto* o = static_cast<__nv_bfloat16*>(p.buf.output);
  auto* res = static_cast<const __nv_bfloat16*>(p.buf.residual);
  constexpr int N = 16 / sizeof(In);
  const bool vec = sh.hidden % 8 == 0 &&
                   ((reinterpret_cast<uintptr_t>(d) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(res)) & 15) == 0;
  auto go = [&](auto kernel, int per_block) {
    launch_pdl(kernel, dim3(sh.tokens, (sh.hidden + per_block - 1) / per_block), dim3(kThreads), 0, s, d,
               static_cast<const int*>(p.buf.mapping), static_cast<const float*>(p.buf.routing_weights), o,
               static_cast<const int*>(p.buf.valid_routes), res, sh.hidden, sh.topk);
  };
  // Unaligned rows, one value per thread while all blocks are resident at once (32 per SM), where latency counts (51 tokens
  // x 247, 8 slots: 6.9 us with one, 7.9 with eight); beyond that launching blocks takes the time (1504 x 799: 22.3 and 5.4 us).
  if (vec) go(combine_kernel<In, true, 1>, kThreads * N);
  else if (static_cast<long long>(sh.tokens) * ((sh.hidden + kThreads - 1) / kThreads) <= 32LL * p.num_sms)
    go(combine_kernel<In, false, 1>, kThreads);
  else
    go(combine_kernel<In, false, 8>, kThreads * 8);
}

}  // namespace

cudaError_t launch_combine(const B200MoePlan& p, cudaStream_t s) {
  if (p.int8) launch_typed<float>(p, s);
  else launch_typed<__nv_bfloat16>(p, s);
  return cudaPeekAtLastError();
}

}  // namespace b200moe
