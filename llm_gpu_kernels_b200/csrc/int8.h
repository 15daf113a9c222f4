// The 8-bit integer kernels behind INT8 plans (abi.cu) and the dense product (linear.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>
#include "../../include/b200moe.h"

namespace b200moe {

constexpr int kInt8MaxK = 131072;   // 127 * 127 * K stays below 2^31

constexpr int int8_pitch(int k) { return (k + 15) / 16 * 16; }   // bytes of a row of int8: TMA strides are multiples of 16

struct QuantizeRows {
  const void* x;
  long long pitch;   // elements
  int dtype;         // B200MOE_BF16 / FP16 / FP32
  int rows, k;
  int8_t* q;         // [rows, int8_pitch(k)]
  float* scale;      // [rows]
  const int* mapping; // null, or [rows * copies]: the rows of q and scale that get row r (16-bit x)
  int copies;
};
cudaError_t launch_quantize_rows(const QuantizeRows& a, cudaStream_t s);

// The dense product for a few tokens (linear_small.cu), which quantises x itself.
struct LinearSmall {
  const void* x;
  long long x_pitch;   // elements
  const int8_t* weight;
  const float* w_scale;
  void* y;
  int8_t* q;           // the quantised rows and their scales, for whoever reads the workspace
  float* q_scale;
  int dtype, tokens, k, n, sms;
};
bool linear_small_serves(int tokens, int k, int n);
cudaError_t launch_linear_small(const LinearSmall& a, cudaStream_t s);

// One of the two products of a layer for a few routes (layer_small.cu), which quantises its rows itself.
struct LayerSmall {
  const void* x;             // gate/up: BF16 rows of the tokens; down: FP32 rows in grouped order
  const int8_t* weight;
  const float* w_scale;
  float* y;                  // [routes, n_out] in grouped order
  int8_t* q;                 // the quantised rows and their scales, for whoever reads the workspace
  float* q_scale;
  const void* ids;
  const int* mapping;
  int ids_are_int64, experts, topk, routes, k, n_out, w_rows;
};
bool layer_small_serves(int tokens, int topk, int hidden, int intermediate);
cudaError_t launch_layer_small(const LayerSmall& a, bool gate_up, int sms, cudaStream_t s);

// One grouped product in int8 (grouped_gemm_i8.cu). Rows of group e are offsets[e] .. + counts[e] of the activations, or
// without `tasks` all `rows` of them belong to the one group there is.
struct I8Gemm {
  CUtensorMap tm_w;            // int8 [groups * w_rows, k], rows int8_pitch(k) bytes apart, box 128 bytes x 128 rows
  CUtensorMap tm_act;          // int8 [rows, k], box 128 bytes x token_tile rows
  const float* w_scale;        // [groups * w_rows]
  const float* row_scale;      // [rows]
  void* out;                   // gate/up: float [rows, n_out]; else [rows, n_out] of out_dtype
  const int* offsets;
  const int* counts;
  const int* tasks;
  int* status;
  int groups, rows, n_out, k, w_rows, token_tile, stages, stream_weights;
  int boxes;                   // tiles of 128 channels per stage (gate/up: 2)
  int split;                   // CTAs of a cluster that share a tile's K; 1: persistent CTAs, a tile each
  int grid;
};
int i8_stages(int out_bytes, int boxes, int token_tile, int split, int* smem_bytes);   // out_bytes: of an output value
// Cycles that a product of `row_tiles` tiles of `token_tile` rows with n_out channels and k values would take in the
// given form, or -1 where the form does not exist. See grouped_gemm_i8.cu.
double i8_cycles(long long row_tiles, int n_out, int k, int token_tile, int boxes, int split, int sms);
int configure_i8();   // opt-in shared memory of the kernels on the current device
cudaError_t launch_i8_gate_up(const I8Gemm& g, cudaStream_t s);
cudaError_t launch_i8_product(const I8Gemm& g, int out_dtype, cudaStream_t s);
// 2-D int8 tensor map, box 128 bytes x box_rows, 128-byte swizzle, zero fill past the ends.
int encode_i8(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t box_rows,
              bool weights);

}  // namespace b200moe
