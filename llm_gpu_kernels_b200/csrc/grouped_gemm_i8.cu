// Ragged grouped product in 8-bit integers on the tensor cores: tcgen05.mma kind::i8, int32 accumulators in tensor
// memory.  y[r, n] = (sum_k q[r, k] W[e, n, k]) * row_scale[r] * w_scale[e, n]  for the rows r of group e.
//
// The organisation is that of the BF16 kernel (grouped_gemm_tcgen05.cu): weights are the M operand (128 output channels
// of a group), rows the N operand, N set per tile; one persistent CTA per SM, warp 0 loads by TMA, warps 1 and 6 issue
// the MMAs of one accumulator each, warps 2-5 drain accumulators, warps 7-10 gather token rows. A k-block is 128 bytes
// = 128 values: the same bytes per stage as there, twice the products. Sums are exact in 32 bits (k <= 131072), so
// neither the tile schedule nor the order of K can change a bit of the result.
//
// gate/up: the two accumulators are the gate and the up rows of the same 128 channels; the epilogue scales both,
// applies SwiGLU and stores FP32: the down product quantises these rows against their largest value, and rounding
// them to BF16 first would move one in a hundred of the 8-bit values to its neighbour (0.8 % of the result).
// product: the two accumulators are two neighbouring tiles of 128 channels (256 channels per tile share every row).
//
// Bound by: HBM while a group has few rows (the weights are streamed once: 604 MB for 128 experts of 2048 x 768, half of
// BF16), by operand bytes through L2 and shared memory beyond.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "gemm_tile.cuh"
#include "int8.h"
#include "pdl.cuh"
#include "plan.h"
#include "sm100_ptx.cuh"

namespace b200moe {
namespace {

using namespace ptx;
using namespace tile;

constexpr int kThreads = 224;
constexpr int kMmaWarpB = 6;
constexpr int kGatherWarps = 4;
constexpr int kGatherThreads = kThreads + 32 * kGatherWarps;
constexpr int kMaxStages = 12;
constexpr int kRowBytes = 128;                       // K bytes of a stage
constexpr uint32_t kBoxBytes = kTileM * kRowBytes;   // one weight box, 16 KB
constexpr uint32_t kWBytes = 2 * kBoxBytes;
constexpr int kCtrlBytes = 4096;
constexpr int kMaxTile = 256;

struct Ctrl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t drain[2];
  uint32_t tmem_base;
  int abort;
  Tables tables;
};
static_assert(sizeof(Ctrl) <= kCtrlBytes, "control block too large");

__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_out(__half* p, float v) { *p = __float2half_rn(v); }

// kGateUp: SwiGLU epilogue (Out = float). kGather: token rows through source_rows.
template <bool kGateUp, bool kGather, typename Out>
__global__ void __launch_bounds__(kGather ? kGatherThreads : kThreads, 1)
grouped_gemm_i8_kernel(const __grid_constant__ I8Gemm g) {
  constexpr int kTileChannels = kGateUp ? kTileM : 2 * kTileM;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Ctrl* c = reinterpret_cast<Ctrl*>(smem_raw);
  const uint32_t raw_addr = smem_u32(smem_raw);
  const uint32_t stage_off = ((raw_addr + kCtrlBytes + 1023u) & ~1023u) - raw_addr;
  unsigned char* stages = smem_raw + stage_off;
  const int token_tile = g.token_tile, num_stages = g.stages;
  const uint32_t stage_bytes = kWBytes + static_cast<uint32_t>(token_tile) * kRowBytes;
  const int acc_cols = 2 * token_tile;
  const int num_acc = 2 * acc_cols <= 512 ? 2 : 1;
  uint32_t tmem_cols = 32;
  while (tmem_cols < static_cast<uint32_t>(num_acc * acc_cols)) tmem_cols <<= 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int E = g.groups;

  if (threadIdx.x == 0) {
    for (int s = 0; s < num_stages; ++s) {
      mbar_init(&c->full[s], kGather ? 1 + 32 * kGatherWarps : 1);
      mbar_init(&c->empty[s], 2);   // the commits of the two MMA issuers
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&c->tmem_full[a], 2);
      mbar_init(&c->tmem_empty[a], 4);   // one arrival per epilogue warp
      mbar_init(&c->drain[a], 1);
    }
    c->abort = 0;
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc(&c->tmem_base, tmem_cols);
  prefetch_head(g.prefetch_base, g.prefetch_chunks);   // HBM is idle while the kernels before this one run
  pdl_wait();
  pdl_launch_dependents();
  if (g.tasks != nullptr) {
    load_tables(&c->tables, g.tasks, g.offsets, g.counts, E);
  } else if (threadIdx.x == 0) {
    c->tables.tasks[0] = 0;
    c->tables.tasks[1] = (g.rows + token_tile - 1) / token_tile;
    c->tables.offsets[0] = 0;
    c->tables.counts[0] = g.rows;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(&c->tmem_base);
  const int n_ct = (g.n_out + kTileChannels - 1) / kTileChannels;
  const int num_kb = (g.k + kRowBytes - 1) / kRowBytes;
  const int total_items = c->tables.tasks[E] * n_ct;

  if (warp == 0) {
    if (lane == 0) {
      // ---------------------------------------------------------------- TMA producer
      const uint64_t pol_w = g.stream_weights ? policy_evict_first() : policy_evict_last();
      const uint64_t pol_act = policy_evict_last();
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
      for (int item = blockIdx.x; ok && item < total_items; item += gridDim.x) {
        const Tile t = decode_tile(&c->tables, item, E, n_ct, token_tile);
        const int w_row = t.expert * g.w_rows + t.ct * kTileChannels;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&c->empty[stage], phase ^ 1u, &c->abort, g.status)) { ok = false; break; }
          unsigned char* st = stages + static_cast<size_t>(stage) * stage_bytes;
          mbar_expect_tx(&c->full[stage], kGather ? kWBytes : stage_bytes);
          tma_load_2d(st, &g.tm_w, &c->full[stage], kb * kRowBytes, w_row, pol_w);
          tma_load_2d(st + kBoxBytes, &g.tm_w, &c->full[stage], kb * kRowBytes, w_row + (kGateUp ? g.n_out : kTileM), pol_w);
          if (!kGather) tma_load_2d(st + kWBytes, &g.tm_act, &c->full[stage], kb * kRowBytes, t.row0, pol_act);
          ++issued;
          if (++stage == num_stages) { stage = 0; phase ^= 1u; }
        }
      }
      // never leave with copies in flight
      const long long first = issued > num_stages ? issued - num_stages : 0;
      for (long long i = first; i < issued; ++i) {
        const int s = static_cast<int>(i % num_stages);
        if (!mbar_wait_plain(&c->full[s], static_cast<uint32_t>((i / num_stages) & 1))) {
          atomicOr(g.status, B200MOE_STATUS_TIMEOUT);
          break;
        }
      }
    }
  } else if (warp == 1 || warp == kMmaWarpB) {
    if (lane == 0) {
      // ---------------------------------------------------------------- MMA issuers (one accumulator each)
      const int half = warp == 1 ? 0 : 1;
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int item = blockIdx.x; ok && item < total_items; item += gridDim.x) {
        const Tile t = decode_tile(&c->tables, item, E, n_ct, token_tile);
        const uint32_t idesc = umma_idesc_i8(kTileM, t.n_eff);
        if (!mbar_wait(&c->tmem_empty[acc], acc_phase ^ 1u, &c->abort, g.status)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * acc_cols + half * token_tile);
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&c->full[stage], phase, &c->abort, g.status)) { ok = false; break; }
          tc_fence_after();
          if (kGather) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // cp.async-written rows -> MMA
          const uint32_t w_addr = smem_u32(stages + static_cast<size_t>(stage) * stage_bytes);
          const uint32_t a_addr = w_addr + kWBytes;
#pragma unroll
          for (int k = 0; k < kRowBytes / 32; ++k)
            umma_i8(d, umma_desc(w_addr + half * kBoxBytes + k * 32), umma_desc(a_addr + k * 32), idesc,
                    (kb | k) != 0 ? 1u : 0u);
          umma_commit(&c->empty[stage]);
          if (++stage == num_stages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit(&c->tmem_full[acc]);
        if (++acc == num_acc) { acc = 0; acc_phase ^= 1u; }
      }
      if (!ok) {   // gave up: let the MMAs already issued finish before TMEM is freed
        umma_commit(&c->drain[half]);
        mbar_wait_plain(&c->drain[half], 0);
      }
    }
  } else if (kGather && warp > kMmaWarpB) {
    // ------------------------------------------------------------------ gather warps: token rows -> activation tile
    constexpr int kIters = kMaxTile * 8 / (32 * kGatherWarps);   // 16-byte pieces per lane and stage
    const int gt = (warp - kMmaWarpB - 1) * 32 + lane;
    const int chunk = gt & 7;
    const int pitch = int8_pitch(g.k);
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < total_items; item += gridDim.x) {
      const Tile t = decode_tile(&c->tables, item, E, n_ct, token_tile);
      const int iters = (t.rows * 8 + 32 * kGatherWarps - 1) / (32 * kGatherWarps);
      int src[kIters];   // token of row it * 16 + gt / 8, -1 past the tile's rows
#pragma unroll
      for (int it = 0; it < kIters; ++it) {
        const int n = it * 16 + (gt >> 3);
        src[it] = (it < iters && n < t.rows) ? g.source_rows[t.row0 + n] : -1;
      }
      for (int kb = 0; kb < num_kb; ++kb) {
        int free_ok = 1;
        if (lane == 0) free_ok = mbar_wait(&c->empty[stage], phase ^ 1u, &c->abort, g.status) ? 1 : 0;
        free_ok = __shfl_sync(0xffffffffu, free_ok, 0);
        if (!free_ok) { ok = false; break; }
        const uint32_t act = smem_u32(stages + static_cast<size_t>(stage) * stage_bytes) + kWBytes;
        const int k = kb * kRowBytes + chunk * 16;
        const uint32_t bytes = k < pitch ? 16u : 0u;   // a piece past the row is zero-filled, as TMA does
#pragma unroll
        for (int it = 0; it < kIters; ++it) {
          if (it < iters && src[it] >= 0) {
            const int n = it * 16 + (gt >> 3);
            const uint32_t dst = act + static_cast<uint32_t>(n) * 128u + (static_cast<uint32_t>(chunk ^ (n & 7)) << 4);
            const int8_t* from = g.x_q + static_cast<size_t>(src[it]) * pitch + (bytes ? k : 0);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
          }
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&c->full[stage])) : "memory");
        if (++stage == num_stages) { stage = 0; phase ^= 1u; }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");   // never leave with copies in flight
  } else {
    // ------------------------------------------------------------------ epilogue warps
    const int quarter = warp & 3;
    Out* out = static_cast<Out*>(g.out);
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int item = blockIdx.x; item < total_items; item += gridDim.x) {
      const Tile t = decode_tile(&c->tables, item, E, n_ct, token_tile);
      const int channel = t.ct * kTileChannels + quarter * 32 + lane;      // of the first accumulator
      const int channel_b = kGateUp ? channel : channel + kTileM;
      const bool ok_a = channel < g.n_out, ok_b = channel_b < g.n_out;
      const float* scales = g.w_scale + static_cast<size_t>(t.expert) * g.w_rows;
      const float sa = ok_a ? scales[channel] : 0.0f;
      const float sb = ok_b ? scales[kGateUp ? g.n_out + channel : channel_b] : 0.0f;
      if (!__all_sync(0xffffffffu, mbar_wait(&c->tmem_full[acc], acc_phase, &c->abort, g.status))) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + static_cast<uint32_t>(acc * acc_cols) + (static_cast<uint32_t>(quarter * 32) << 16);
      Out* dst = out + static_cast<size_t>(t.row0) * g.n_out;
      for (int n0 = 0; n0 < t.n_eff; n0 += 16) {
        uint32_t a[16], b[16];
        tmem_ld16(taddr + n0, a);
        tmem_ld16(taddr + token_tile + n0, b);
        // lane j holds the scale of row n0 + j
        const int n_mine = n0 + (lane & 15);
        float row_scale = 0.0f;
        if (n_mine < t.rows) row_scale = g.row_scale[kGather ? g.source_rows[t.row0 + n_mine] : t.row0 + n_mine];
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int n = n0 + j;
          const float s = __shfl_sync(0xffffffffu, row_scale, j);
          const float va = static_cast<float>(static_cast<int>(a[j])) * (s * sa);
          const float vb = static_cast<float>(static_cast<int>(b[j])) * (s * sb);
          if (n < t.rows) {
            Out* row = dst + static_cast<size_t>(n) * g.n_out;
            if (kGateUp) {
              if (ok_a) store_out(row + channel, (va / (1.0f + __expf(-va))) * vb);
            } else {
              if (ok_a) store_out(row + channel, va);
              if (ok_b) store_out(row + channel_b, vb);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&c->tmem_empty[acc]);
      if (++acc == num_acc) { acc = 0; acc_phase ^= 1u; }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, tmem_cols);
  }
}

template <bool kGateUp, bool kGather, typename Out>
cudaError_t launch(const I8Gemm& g, int grid, cudaStream_t s) {
  int smem = 0;
  i8_stages(g.token_tile, &smem);
  return launch_pdl(grouped_gemm_i8_kernel<kGateUp, kGather, Out>, dim3(grid), dim3(kGather ? kGatherThreads : kThreads),
                    smem, s, g);
}

}  // namespace

int i8_stages(int token_tile, int* smem_bytes) {
  const int stage = static_cast<int>(kWBytes) + token_tile * kRowBytes;
  int stages = (kSmemLimit - kCtrlBytes - 1024) / stage;
  if (stages > kMaxStages) stages = kMaxStages;
  *smem_bytes = kCtrlBytes + 1024 + stages * stage;
  return stages;
}

int configure_i8() {
  const void* kernels[] = {reinterpret_cast<const void*>(grouped_gemm_i8_kernel<true, false, float>),
                           reinterpret_cast<const void*>(grouped_gemm_i8_kernel<true, true, float>),
                           reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, false, __nv_bfloat16>),
                           reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, false, __half>)};
  for (const void* kernel : kernels) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (e != cudaSuccess) {
      set_error("cudaFuncSetAttribute(int8 shared memory) failed: %s", cudaGetErrorString(e));
      return B200MOE_ERR_CUDA;
    }
  }
  return B200MOE_OK;
}

cudaError_t launch_i8_gate_up(const I8Gemm& g, bool gather, int grid, cudaStream_t s) {
  return gather ? launch<true, true, float>(g, grid, s) : launch<true, false, float>(g, grid, s);
}

cudaError_t launch_i8_product(const I8Gemm& g, int out_dtype, int grid, cudaStream_t s) {
  return out_dtype == B200MOE_FP16 ? launch<false, false, __half>(g, grid, s)
                                   : launch<false, false, __nv_bfloat16>(g, grid, s);
}

}  // namespace b200moe
