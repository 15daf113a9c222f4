// Ragged grouped product in 8-bit integers on the tensor cores: tcgen05.mma kind::i8, int32 accumulators in tensor
// memory.  y[r, n] = (sum_k q[r, k] W[e, n, k]) * row_scale[r] * w_scale[e, n]  for the rows r of group e.
//
// The organisation is that of the BF16 kernel (grouped_gemm_tcgen05.cu): weights are the M operand (128 output channels
// of a group), rows the N operand, N set per tile; one persistent CTA per SM, warp 0 loads by TMA, warps 1 and 6 issue
// the MMAs of one accumulator each, warps 2-5 and 7-10 drain accumulators. A k-block is 128 bytes = 128 values: the same
// bytes per stage as there, twice the products. Sums are exact in 32 bits (k <= 131072), so neither the tile schedule nor
// the order of K can change a bit of the result. Token rows are not gathered here: the kernel that quantises x writes
// them in grouped order, one byte per value, and a TMA box brings them (gathering them in four warps with cp.async, as
// the BF16 kernel does: 156 and 151 us for 1024 tokens of 128 experts, 348 and 300 for 4096, 110 and 102 for 193 of 60).
//
// gate/up: the two accumulators are the gate and the up rows of the same 128 channels; the epilogue scales both,
// applies SwiGLU and stores FP32: the down product quantises these rows against their largest value, and rounding
// them to BF16 first would move one in a hundred of the 8-bit values to its neighbour (normal gate and up: 1.6 % of them
// at 768 channels, 1.0 % at 14336, by which the result moves 0.8 and 1.0 %). The rows of
// a layer's down product stay FP32 as well, until the combine has summed them: the result is rounded once. As BF16 rows
// they made a layer's error against 64 bits 0.0024 of the result instead of 0.0017, and saved a twentieth of its time at
// most (1024 tokens of 128 experts 152.3 us, with FP32 rows 159.6; 2048 of 8 large ones 852 and 871).
// product: the two accumulators are two neighbouring tiles of 128 channels (256 channels per tile share every row), or
// with one box per stage the even and the odd K steps of one tile of 128 channels, added in the epilogue.
//
// Epilogue: the accumulator has the channel on the lane, so a warp that stored what it holds would write 64 bytes of each
// row per instruction, two per lane. It passes 16 rows of its 32 channels through 2 KB of shared memory of its own and
// writes 16 bytes per lane. Eight warps share the work: with 256-row tiles the accumulators take all of tensor memory
// and nothing hides the epilogue.
//
// kSplit: few tiles for the SMs there are. A thread-block cluster works on one tile, each CTA on a slice of K; the
// int32 partial sums meet through distributed shared memory (exact, so the split changes no bit either) and every CTA
// finishes some of the rows.
//
// The kernel in front of this one (int8_quant.cu) lets its dependents start only after its own wait, so everything before
// IT is complete and visible when this kernel starts: the dispatch's tables and the weights may be read at once, and
// the first stages of weights are on their way while the rows are still being quantised. Only the rows, their scales
// and the output wait.
//
// Bound by: HBM while a group has few rows (the weights are streamed once: 604 MB for 128 experts of 2048 x 768, half of
// BF16; with 64 rows each gate/up takes 80 us and reads 5.3 TB/s, the down product, which writes 67 MB of FP32 rows, 44 us;
// the last round of tiles fills a fifth of the SMs), by operand bytes through L2 and shared memory beyond (8192 x 4096 x
// 14336: 337 us in a short burst, 2.86 POP/s, tensor pipe busy 72 % of its cycles; 404 us for seconds under the power limit).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>
#include "gemm_tile.cuh"
#include "int8.h"
#include "int8_rows.cuh"
#include "pdl.cuh"
#include "plan.h"
#include "sm100_ptx.cuh"

namespace b200moe {
namespace {

using namespace ptx;
using namespace tile;

constexpr int kThreads = 224;   // warps 0 .. 6
constexpr int kMmaWarpB = 6;
constexpr int kMaxThreads = kThreads + 32 * 4;   // warps 7-10 drain accumulators as warps 2-5 do
constexpr int kMaxStages = 12;
constexpr int kRowBytes = 128;                       // K bytes of a stage
constexpr uint32_t kBoxBytes = kTileM * kRowBytes;   // one weight box, 16 KB
constexpr int kCtrlBytes = 4096;
constexpr int kMaxTile = 256;
constexpr int kMaxSplit = 8;

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

// What an epilogue warp has in shared memory, behind Ctrl.
template <typename Out>
struct EpilogueWarp {
  static constexpr int kPitch = 32 * sizeof(Out) + 16;   // padding against bank conflicts
  alignas(16) float row_scale[kMaxTile];                 // of the tile it works on
  alignas(16) unsigned char transpose[16 * kPitch];      // 16 rows of its 32 channels
};
constexpr int kEpilogueWarps = 8;   // two teams of four, one warp per quarter of the TMEM lanes
// Ctrl, and behind it what the epilogue needs: an EpilogueWarp each, or the row scales of a split tile.
__host__ __device__ constexpr int ctrl_bytes(int out_bytes, bool split) {
  return kCtrlBytes + (split ? kMaxTile * 4
                             : kEpilogueWarps * static_cast<int>(out_bytes == 4 ? sizeof(EpilogueWarp<float>) : sizeof(EpilogueWarp<__half>)));
}

// Rows 0 .. 15 (of which `rows` exist) of 32 channels from channel0: v[j] is row j of channel channel0 + lane. `dst` is
// row 0; `buffer` is this warp's own. Rows that start on 16 bytes are written in pieces of 16 bytes.
template <typename Out>
__device__ __forceinline__ void store_rows(Out* dst, const float (&v)[16], int rows, int channel0, int n_out,
                                           unsigned char* buffer, int lane) {
  constexpr int kTransposePitch = EpilogueWarp<Out>::kPitch;
  constexpr int kPiece = 16 / sizeof(Out), kPerRow = 32 / kPiece;   // values per piece, pieces per row
  if (n_out % kPiece == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
    __syncwarp();   // the rows before are read
#pragma unroll
    for (int j = 0; j < 16; ++j) store_out(reinterpret_cast<Out*>(buffer + j * kTransposePitch) + lane, v[j]);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16 * kPerRow / 32; ++i) {
      const int row = i * (32 / kPerRow) + lane / kPerRow, channel = channel0 + (lane % kPerRow) * kPiece;
      const uint4 piece = *reinterpret_cast<const uint4*>(buffer + row * kTransposePitch + (lane % kPerRow) * 16);
      if (row < rows && channel < n_out) *reinterpret_cast<uint4*>(dst + static_cast<size_t>(row) * n_out + channel) = piece;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < rows && channel0 + lane < n_out) store_out(dst + static_cast<size_t>(j) * n_out + channel0 + lane, v[j]);
  }
}

// kFar: some products of two scales of the tile may be out of range; see rows8::scaled.
template <bool kFar>
__device__ __forceinline__ float scaled(uint32_t sum, float row, float channel) {
  return kFar ? rows8::scaled(static_cast<int>(sum), row, channel) : static_cast<float>(static_cast<int>(sum)) * (row * channel);
}
// Four channels of a row; out of line, for the same reason.
__device__ __noinline__ float4 scaled_far4(int4 sum, float row, float4 channel) {
  return make_float4(rows8::scaled(sum.x, row, channel.x), rows8::scaled(sum.y, row, channel.y),
                     rows8::scaled(sum.z, row, channel.z), rows8::scaled(sum.w, row, channel.w));
}
// The smallest and the largest finite scale above 0 of some rows, as bits.
struct RowScales {
  uint32_t least = 0x7f800000u, most = 0u;
  __device__ __forceinline__ void add(float s) {
    if (s > 0.0f && s < INFINITY) {
      least = min(least, __float_as_uint(s));
      most = max(most, __float_as_uint(s));
    }
  }
  __device__ __forceinline__ void join() {   // those of the warp's lanes
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
  }
  __device__ __forceinline__ bool far(float channel) const {
    return channel != 0.0f && most != 0u && !(rows8::in_range(__uint_as_float(least) * channel) && rows8::in_range(__uint_as_float(most) * channel));
  }
};
// __expf: within 2^-22 + |gate| 2^-23, a thousandth of the step of 1 / 127 that the row is rounded to next.
__device__ __forceinline__ float swiglu(float gate, float up) { return (gate / (1.0f + __expf(-gate))) * up; }

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int4 ld_cluster_int4(uint32_t addr, uint32_t cta) {
  uint32_t remote;
  int4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(cta));
  asm volatile("ld.shared::cluster.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(remote));
  return v;
}

// kGateUp: SwiGLU epilogue (Out = float, two boxes). kBoxes: weight boxes (tiles of 128 channels) per stage. kSplit: one
// tile per cluster, K split over its CTAs.
template <bool kGateUp, int kBoxes, bool kSplit, typename Out>
__global__ void __launch_bounds__(kMaxThreads, 1)
grouped_gemm_i8_kernel(const __grid_constant__ I8Gemm g) {
  static_assert(!kGateUp || kBoxes == 2, "gate and up are the two boxes");
  constexpr int kTileChannels = kGateUp ? kTileM : kBoxes * kTileM;
  constexpr uint32_t kWBytes = kBoxes * kBoxBytes;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Ctrl* c = reinterpret_cast<Ctrl*>(smem_raw);
  const uint32_t raw_addr = smem_u32(smem_raw);
  constexpr uint32_t kCtrl = ctrl_bytes(sizeof(Out), kSplit);
  const uint32_t stage_off = ((raw_addr + kCtrl + 1023u) & ~1023u) - raw_addr;
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
      mbar_init(&c->full[s], 1);
      mbar_init(&c->empty[s], 2);   // the commits of the two MMA issuers
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&c->tmem_full[a], 2);
      mbar_init(&c->tmem_empty[a], kEpilogueWarps);   // one arrival each
      mbar_init(&c->drain[a], 1);
    }
    c->abort = 0;
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc(&c->tmem_base, tmem_cols);
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
  // the tiles of this CTA and the K blocks it does of them
  int first_item = blockIdx.x, item_step = gridDim.x, kb0 = 0, kb1 = num_kb;
  uint32_t cta = 0, ctas = 1;
  if (kSplit) {   // one tile per cluster, a slice of its K blocks per CTA
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(cta));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
    const int per = (num_kb + static_cast<int>(ctas) - 1) / static_cast<int>(ctas);
    kb0 = min(num_kb, static_cast<int>(cta) * per);
    kb1 = min(num_kb, kb0 + per);
    first_item = kb0 < kb1 ? blockIdx.x / ctas : total_items;
    item_step = total_items;
  }
  const bool any = first_item < total_items;
  float* split_rows = reinterpret_cast<float*>(smem_raw + kCtrlBytes);   // the row scales of a split tile
  auto next_item = [&](int item) { return total_items - item > item_step ? item + item_step : total_items; };

  if (warp == 0) {
    if (lane == 0) {
      // ---------------------------------------------------------------- TMA producer
      const uint64_t pol_w = g.stream_weights ? policy_evict_first() : policy_evict_last();
      const uint64_t pol_act = policy_evict_last();
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
      auto load_weights = [&](const Tile& t, int kb, int st) {
        unsigned char* to = stages + static_cast<size_t>(st) * stage_bytes;
        const int w_row = t.expert * g.w_rows + t.ct * kTileChannels;
        mbar_expect_tx(&c->full[st], stage_bytes);
        tma_load_2d(to, &g.tm_w, &c->full[st], kb * kRowBytes, w_row, pol_w);
        if (kBoxes == 2)
          tma_load_2d(to + kBoxBytes, &g.tm_w, &c->full[st], kb * kRowBytes, w_row + (kGateUp ? g.n_out : kTileM), pol_w);
      };
      int early = 0;   // stages of the first tile whose weights are already on their way
      if (any) {
        const Tile t = decode_tile(&c->tables, first_item, E, n_ct, token_tile);
        for (; early < num_stages && kb0 + early < kb1; ++early) load_weights(t, kb0 + early, early);
      }
      pdl_wait();
      for (int item = first_item; ok && item < total_items; item = next_item(item)) {
        const Tile t = decode_tile(&c->tables, item, E, n_ct, token_tile);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (early > 0) {
            --early;
          } else {
            if (!mbar_wait(&c->empty[stage], phase ^ 1u, &c->abort, g.status)) { ok = false; break; }
            load_weights(t, kb, stage);
          }
          tma_load_2d(stages + static_cast<size_t>(stage) * stage_bytes + kWBytes, &g.tm_act, &c->full[stage], kb * kRowBytes,
                      t.row0, pol_act);
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
      for (int item = first_item; ok && item < total_items; item = next_item(item)) {
        const Tile t = decode_tile(&c->tables, item, E, n_ct, token_tile);
        const uint32_t idesc = umma_idesc_i8(kTileM, t.n_eff);
        if (!mbar_wait(&c->tmem_empty[acc], acc_phase ^ 1u, &c->abort, g.status)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * acc_cols + half * token_tile);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&c->full[stage], phase, &c->abort, g.status)) { ok = false; break; }
          tc_fence_after();
          const uint32_t w_addr = smem_u32(stages + static_cast<size_t>(stage) * stage_bytes);
          const uint32_t a_addr = w_addr + kWBytes;
#pragma unroll
          for (int k = 0; k < kRowBytes / 32; ++k) {
            if (kBoxes == 2)
              umma_i8(d, umma_desc(w_addr + half * kBoxBytes + k * 32), umma_desc(a_addr + k * 32), idesc,
                      kb != kb0 || k != 0 ? 1u : 0u);
            else if ((k & 1) == half)
              umma_i8(d, umma_desc(w_addr + k * 32), umma_desc(a_addr + k * 32), idesc, kb != kb0 || k > 1 ? 1u : 0u);
          }
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
  } else {
    // ------------------------------------------------------------------ epilogue warps
    const int quarter = warp & 3;                      // the TMEM lane quarter this warp may read
    const int team = warp < kMmaWarpB ? 0 : 1;         // of the two warps of a quarter
    EpilogueWarp<Out>* mine = reinterpret_cast<EpilogueWarp<Out>*>(smem_raw + kCtrlBytes) + team * 4 + quarter;
    int acc = 0;
    uint32_t acc_phase = 0;
    if (!kSplit) pdl_wait();   // row scales and output
    if constexpr (kSplit) {
      const int tile = blockIdx.x / ctas;   // also of a CTA without K blocks: it finishes rows
      if (tile < total_items) {
        const Tile t = decode_tile(&c->tables, tile, E, n_ct, token_tile);
        pdl_wait();
        for (int n = (team * 4 + quarter) * 32 + lane; n < t.rows; n += kEpilogueWarps * 32) split_rows[n] = g.row_scale[t.row0 + n];
      }
    }
    for (int item = first_item; item < total_items; item = next_item(item)) {
      const Tile t = decode_tile(&c->tables, item, E, n_ct, token_tile);
      const int channel = t.ct * kTileChannels + quarter * 32 + lane;      // of the first box
      const int channel_b = kGateUp ? channel : channel + kTileM;
      const bool ok_a = channel < g.n_out, ok_b = kBoxes == 2 && channel_b < g.n_out;
      const float* scales = g.w_scale + static_cast<size_t>(t.expert) * g.w_rows;
      const float sa = !kSplit && ok_a ? scales[channel] : 0.0f;
      const float sb = !kSplit && ok_b ? scales[kGateUp ? g.n_out + channel : channel_b] : 0.0f;
      // the tile's row scales while its MMAs still run: fetched chunk by chunk they cost two L2 round trips per 16 rows
      float* row_scale = mine->row_scale;
      bool far = false;
      if constexpr (!kSplit) {
        RowScales scales_here;
        for (int n = lane; n < t.n_eff; n += 32) {
          const float s = n < t.rows ? g.row_scale[t.row0 + n] : 0.0f;
          row_scale[n] = s;
          scales_here.add(s);
        }
        scales_here.join();
        far = __any_sync(0xffffffffu, scales_here.far(sa) || scales_here.far(sb));
      }
      if (!__all_sync(0xffffffffu, mbar_wait(&c->tmem_full[acc], acc_phase, &c->abort, g.status))) break;
      __syncwarp();
      tc_fence_after();
      const uint32_t taddr = tmem_base + static_cast<uint32_t>(acc * acc_cols) + (static_cast<uint32_t>(quarter * 32) << 16);
      if (kSplit) {
        // partial sums [box][row][128], for the cluster, into the drained stages
        int* part = reinterpret_cast<int*>(stages) + quarter * 32 + lane;
        for (int n0 = team * 16; n0 < t.n_eff; n0 += 32) {
          uint32_t a[16], b[16];
          tmem_ld16(taddr + n0, a);
          tmem_ld16(taddr + token_tile + n0, b);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            part[(n0 + j) * kTileM] = static_cast<int>(kBoxes == 2 ? a[j] : a[j] + b[j]);
            if (kBoxes == 2) part[(token_tile + n0 + j) * kTileM] = static_cast<int>(b[j]);
          }
        }
      } else {
        Out* dst = static_cast<Out*>(g.out) + static_cast<size_t>(t.row0) * g.n_out;
        // this team's part: one of the two boxes, or every other 16 rows
        constexpr bool kByBox = !kGateUp && kBoxes == 2;
        auto drain = [&](auto far_scales) {
          constexpr bool kFar = decltype(far_scales)::value;
          for (int n0 = kByBox ? 0 : team * 16; n0 < t.n_eff; n0 += kByBox ? 16 : 32) {
            uint32_t a[16], b[16];
            if (kByBox) {
              tmem_ld16(taddr + (team ? token_tile : 0) + n0, a);
            } else {
              tmem_ld16(taddr + n0, a);
              tmem_ld16(taddr + token_tile + n0, b);
            }
            float scale[16];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<float4*>(scale + 4 * j) = *reinterpret_cast<const float4*>(row_scale + n0 + 4 * j);
            tmem_ld_wait();
            float v[16];
            [[maybe_unused]] const float s_mine = kByBox && team ? sb : sa;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              if constexpr (kGateUp) v[j] = swiglu(scaled<kFar>(a[j], scale[j], sa), scaled<kFar>(b[j], scale[j], sb));
              else if constexpr (kBoxes == 1) v[j] = scaled<kFar>(a[j] + b[j], scale[j], sa);
              else v[j] = scaled<kFar>(a[j], scale[j], s_mine);
            }
            const int channel0 = (kByBox && team ? channel_b : channel) - lane;
            store_rows(dst + static_cast<size_t>(n0) * g.n_out, v, t.rows - n0, channel0, g.n_out, mine->transpose, lane);
          }
        };
        if (far) drain(std::true_type{});
        else drain(std::false_type{});
      }
      tc_fence_before();
      __syncwarp();   // also: row_scale is read before the next tile's is written
      if (lane == 0) mbar_arrive(&c->tmem_empty[acc]);
      if (++acc == num_acc) { acc = 0; acc_phase ^= 1u; }
    }
  }

  if constexpr (kSplit) {
    // ------------------------------------------------------------------ the cluster's partial sums -> output
    __syncwarp();
    cluster_barrier();   // every CTA's partial sums are in its shared memory
    pdl_wait();          // output
    const int tile = blockIdx.x / ctas;
    if (tile < total_items && !*reinterpret_cast<volatile int*>(&c->abort)) {
      const Tile t = decode_tile(&c->tables, tile, E, n_ct, token_tile);
      const int per = (num_kb + static_cast<int>(ctas) - 1) / static_cast<int>(ctas);
      const int active = (num_kb + per - 1) / per;   // CTAs that had K blocks
      const uint32_t base = smem_u32(stages) + static_cast<uint32_t>(lane) * 16u;
      Out* dst = static_cast<Out*>(g.out) + static_cast<size_t>(t.row0) * g.n_out;
      // the scales of this lane's four channels, of gate and up or of both boxes
      const float* scales = g.w_scale + static_cast<size_t>(t.expert) * g.w_rows;
      float split_scale[kBoxes][4] = {};
#pragma unroll
      for (int b = 0; b < kBoxes; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int channel = t.ct * kTileChannels + (kGateUp ? 0 : b * kTileM) + lane * 4 + j;
          if (channel < g.n_out) split_scale[b][j] = scales[kGateUp ? b * g.n_out + channel : channel];
        }
      // Each CTA finishes every ctas-th row, a warp two vectors of 4 channels x 32 lanes at a time: gate and up of a row,
      // its two boxes, or with one box two rows. All loads of the two come first: one round trip through the cluster.
      constexpr int kRows = kBoxes == 2 ? 1 : 2;
      const int stride = static_cast<int>(ctas) * kMaxThreads / 32;
      for (int n = static_cast<int>(cta) + static_cast<int>(ctas) * warp; n < t.rows; n += kRows * stride) {
        int4 v[2][kMaxSplit];
        const int vectors = kRows == 2 && n + stride >= t.rows ? 1 : 2;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int at = kRows == 2 ? n + b * stride : b * token_tile + n;
#pragma unroll
          for (int i = 0; i < kMaxSplit; ++i)
            if (i < active && b < vectors) v[b][i] = ld_cluster_int4(base + static_cast<uint32_t>(at * kTileM * 4), i);
        }
        float y[2][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          int sum[4] = {};
#pragma unroll
          for (int i = 0; i < kMaxSplit; ++i)
            if (i < active) {
              sum[0] += v[b][i].x; sum[1] += v[b][i].y; sum[2] += v[b][i].z; sum[3] += v[b][i].w;
            }
          const float row_scale = split_rows[kRows == 2 ? min(n + b * stride, t.rows - 1) : n];
          const float (&channel_scale)[4] = split_scale[kRows == 2 ? 0 : b];
          float least = INFINITY, most = 0.0f;   // NaN passes: its products are NaN either way
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float scale = row_scale * channel_scale[j];
            y[b][j] = static_cast<float>(sum[j]) * scale;
            least = fminf(least, fabsf(scale));
            most = fmaxf(most, fabsf(scale));
          }
          if (!(least >= 0x1p-126f && most < INFINITY)) {
            const float4 far = scaled_far4(make_int4(sum[0], sum[1], sum[2], sum[3]), row_scale,
                                           make_float4(channel_scale[0], channel_scale[1], channel_scale[2], channel_scale[3]));
            y[b][0] = far.x; y[b][1] = far.y; y[b][2] = far.z; y[b][3] = far.w;
          }
        }
#pragma unroll
        for (int b = 0; b < (kGateUp ? 1 : 2); ++b) {
          const int row = kRows == 2 ? n + b * stride : n;
          const int channel = t.ct * kTileChannels + (kRows == 2 ? 0 : b * kTileM) + lane * 4;
          if (row >= t.rows) break;
          Out* to = dst + static_cast<size_t>(row) * g.n_out + channel;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (channel + j < g.n_out) store_out(to + j, kGateUp ? swiglu(y[0][j], y[1][j]) : y[b][j]);
        }
      }
    }
    __syncwarp();
    cluster_barrier();   // no CTA leaves while another may read its shared memory
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem_base, tmem_cols);
  }
}

template <bool kGateUp, int kBoxes, bool kSplit, typename Out>
cudaError_t launch(const I8Gemm& g, cudaStream_t s) {
  int smem = 0;
  i8_stages(sizeof(Out), g.boxes, g.token_tile, g.split, &smem);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(g.grid);
  cfg.blockDim = dim3(kMaxThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = g.split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kSplit ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, grouped_gemm_i8_kernel<kGateUp, kBoxes, kSplit, Out>, g);
}

template <typename Out>
cudaError_t launch_product(const I8Gemm& g, cudaStream_t s) {
  if (g.split > 1) return g.boxes == 2 ? launch<false, 2, true, Out>(g, s) : launch<false, 1, true, Out>(g, s);
  return g.boxes == 2 ? launch<false, 2, false, Out>(g, s) : launch<false, 1, false, Out>(g, s);
}

}  // namespace

int i8_stages(int out_bytes, int boxes, int token_tile, int split, int* smem_bytes) {
  const int stage = boxes * static_cast<int>(kBoxBytes) + token_tile * kRowBytes;
  // the partial sums of a split tile take the place of the drained stages
  const int partial = split > 1 ? boxes * token_tile * kTileM * 4 : 0;
  const int ctrl = ctrl_bytes(out_bytes, split > 1) + 1024;
  int stages = (kSmemLimit - ctrl) / stage;
  if (stages > kMaxStages) stages = kMaxStages;
  *smem_bytes = ctrl + (stages * stage > partial ? stages * stage : partial);
  return stages;
}

// What decides between tile shapes: an estimate that has to rank them, not to tell the time. Its figures were fitted to 33
// timings of 9 to 2048 rows (k 1999 to 4096, n 1536 to 5003) of an earlier form of the kernel, those of the epilogue with one
// set of accumulators and of a split tile again when these changed, to the timings given here. A stage takes the longest of its bytes at 50 bytes per cycle out of L2, its MMAs (half a
// cycle per row and K step of 32) and 210 cycles of hand-over; a tile that is not followed by another on its SM shows
// its epilogue, 36 cycles per row and box; adding up a split tile takes 3200 cycles and 26 per row and box. Above 512
// columns of accumulators there is only one set and every epilogue shows, at 30 cycles per row and box with eight warps:
// 128 x 2 boxes is faster while K is short (8192 x 1024 x 4096: 54 and 66 us), 256 x 2 once K is long, where the power
// limit decides and a third less goes through L2 (8192 x 4096 x 14336, back to back for seconds: 442 and 421 us).
double i8_cycles(long long row_tiles, int n_out, int k, int token_tile, int boxes, int split, int sms) {
  const long long tiles = row_tiles * ((n_out + 128 * boxes - 1) / (128 * boxes));
  const int blocks = (k + kRowBytes - 1) / kRowBytes;
  int smem = 0;
  if (i8_stages(4, boxes, token_tile, split, &smem) < 2 || smem > kSmemLimit) return -1.0;
  const double bytes = boxes * static_cast<double>(kBoxBytes) + token_tile * kRowBytes;
  double block = bytes / 50.0;
  if (block < boxes * 2.0 * token_tile) block = boxes * 2.0 * token_tile;
  if (block < 210.0) block = 210.0;
  const double rows = static_cast<double>(token_tile) * boxes;
  if (split > 1) {
    // All clusters have to be resident at once: pairs take every SM, clusters of 4 leave out two SMs of a GPC, of 8 there
    // are two in most GPCs but not in all (128 rows x 8192 x 1024: 16 clusters of 8 18.5 us, half as many CTAs 13.6).
    if (tiles * split > (split == 8 ? sms * 2 / 3 : split == 4 ? sms * 7 / 8 : sms) || blocks < 2 * split) return -1.0;
    return (blocks + split - 1) / split * block + 3200.0 + 26.0 * rows;
  }
  const double rounds = static_cast<double>((tiles + sms - 1) / sms);
  if (rounds > 1 && 4 * token_tile > 512) return rounds * (blocks * block + 30.0 * rows);
  return rounds * blocks * block + 36.0 * rows;
}

int configure_i8() {
  using bf16 = __nv_bfloat16;
  const void* kernels[] = {
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<true, 2, false, float>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<true, 2, true, float>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 1, false, float>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 1, true, float>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 2, false, float>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 2, true, float>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 1, false, bf16>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 1, true, bf16>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 2, false, bf16>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 2, true, bf16>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 1, false, __half>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 1, true, __half>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 2, false, __half>),
      reinterpret_cast<const void*>(grouped_gemm_i8_kernel<false, 2, true, __half>)};
  for (const void* kernel : kernels) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (e != cudaSuccess) {
      set_error("cudaFuncSetAttribute(int8 shared memory) failed: %s", cudaGetErrorString(e));
      return B200MOE_ERR_CUDA;
    }
  }
  return B200MOE_OK;
}

cudaError_t launch_i8_gate_up(const I8Gemm& g, cudaStream_t s) {
  return g.split > 1 ? launch<true, 2, true, float>(g, s) : launch<true, 2, false, float>(g, s);
}

cudaError_t launch_i8_product(const I8Gemm& g, int out_dtype, cudaStream_t s) {
  if (out_dtype == B200MOE_FP32) return launch_product<float>(g, s);
  return out_dtype == B200MOE_FP16 ? launch_product<__half>(g, s) : launch_product<__nv_bfloat16>(g, s);
}

}  // namespace b200moe
