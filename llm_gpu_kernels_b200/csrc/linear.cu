// One dense product in 8-bit integers behind b200moe_linear_*: quantise the rows of x (int8_quant.cu), then the grouped
// product with a single group (grouped_gemm_i8.cu).
#include <new>
#include "int8.h"
#include "plan.h"

struct B200MoeLinear {
  B200MoeLinearShape shape{};
  B200MoeLinearBuffers buf{};
  bool bound = false;
  bool small = false;   // a few tokens: one kernel without tensor cores
  int token_tile = 16, boxes = 1, split = 1, sms = 0;
  b200moe::I8Gemm gemm{};
};

namespace b200moe {
namespace {

constexpr int kSms = 148;   // B200; the schedule is chosen before a device is touched

// Tile rows, boxes and K split with the least estimated time.
void choose_tiles(B200MoeLinear* p) {
  const B200MoeLinearShape& s = p->shape;
  double best = -1.0;
  for (int boxes = 1; boxes <= 2; ++boxes)
    for (int tile = 16; tile <= 256 && (tile == 16 || tile - 16 < s.tokens); tile += 16)
      for (int split = 1; split <= 8; split *= 2) {
        const double c = i8_cycles((s.tokens + tile - 1) / tile, s.n, s.k, tile, boxes, split, kSms);
        if (c >= 0.0 && (best < 0.0 || c < best)) {
          best = c;
          p->token_tile = tile;
          p->boxes = boxes;
          p->split = split;
        }
      }
}

}  // namespace
}  // namespace b200moe

using namespace b200moe;

extern "C" {

int b200moe_linear_create(const B200MoeLinearShape* shape, B200MoeLinear** out) {
  if (!shape || !out) {
    set_error("null argument");
    return B200MOE_ERR_INVALID;
  }
  if (shape->tokens < 0 || shape->k < 1 || shape->k > kInt8MaxK || shape->n < 1 || shape->n > (1 << 30)) {
    set_error("linear: needs T >= 0, k in [1,%d], n >= 1 (T=%d k=%d n=%d)", kInt8MaxK, shape->tokens, shape->k, shape->n);
    return B200MOE_ERR_INVALID;
  }
  if (shape->dtype != B200MOE_BF16 && shape->dtype != B200MOE_FP16) {
    set_error("linear: x must be BF16 or FP16 (dtype %d)", shape->dtype);
    return B200MOE_ERR_INVALID;
  }
  const long long tiles = (static_cast<long long>(shape->tokens) + 15) / 16 * ((static_cast<long long>(shape->n) + 255) / 256);
  if (tiles >= (1LL << 31) - 1024 || shape->tokens > (1 << 30)) {
    set_error("linear: T=%d x n=%d is too large", shape->tokens, shape->n);
    return B200MOE_ERR_INVALID;
  }
  B200MoeLinear* p = new (std::nothrow) B200MoeLinear();
  if (!p) {
    set_error("out of host memory");
    return B200MOE_ERR_INVALID;
  }
  p->shape = *shape;
  p->small = linear_small_serves(shape->tokens, shape->k, shape->n);
  choose_tiles(p);
  *out = p;
  return B200MOE_OK;
}

int b200moe_linear_workspace(const B200MoeLinear* p, B200MoeLinearWorkspace* w) {
  if (!p || !w) {
    set_error("null argument");
    return B200MOE_ERR_INVALID;
  }
  *w = B200MoeLinearWorkspace{};
  w->x_q = static_cast<size_t>(p->shape.tokens) * int8_pitch(p->shape.k);
  w->x_scale = static_cast<size_t>(p->shape.tokens) * 4;
  w->status = 4;
  w->launches = p->shape.tokens == 0 ? 0 : p->small ? 1 : 2;
  return B200MOE_OK;
}

int b200moe_linear_bind(B200MoeLinear* p, const B200MoeLinearBuffers* b) {
  if (!p || !b) {
    set_error("null argument");
    return B200MOE_ERR_INVALID;
  }
  p->bound = false;
  const B200MoeLinearShape& s = p->shape;
  p->buf = *b;
  if (s.tokens == 0) {
    p->bound = true;
    return B200MOE_OK;
  }
  const void* needed[] = {b->x, b->weight, b->weight_scale, b->output, b->x_q, b->x_scale, b->status};
  for (const void* ptr : needed)
    if (!ptr) {
      set_error("linear: null buffer");
      return B200MOE_ERR_INVALID;
    }
  const void* read[] = {b->x, b->weight, b->weight_scale};
  const void* written[] = {b->output, b->x_q, b->x_scale, b->status};
  for (const void* in : read)
    for (const void* to : written)
      if (in == to) {
        set_error("linear: a written buffer aliases an input");
        return B200MOE_ERR_INVALID;
      }
  if (s.tokens > 1 && b->x_pitch < s.k) {
    set_error("linear: row pitch %lld of x is smaller than k=%d", static_cast<long long>(b->x_pitch), s.k);
    return B200MOE_ERR_INVALID;
  }
  if ((reinterpret_cast<uintptr_t>(b->weight) | reinterpret_cast<uintptr_t>(b->x_q)) % 16 ||
      (reinterpret_cast<uintptr_t>(b->x) | reinterpret_cast<uintptr_t>(b->output)) % 2 ||
      (reinterpret_cast<uintptr_t>(b->weight_scale) | reinterpret_cast<uintptr_t>(b->x_scale) |
       reinterpret_cast<uintptr_t>(b->status)) % 4) {
    set_error("linear: misaligned buffer (weight and x_q 16 bytes, x and output 2, scales and status 4)");
    return B200MOE_ERR_INVALID;
  }
  int device = 0, major = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) {
    set_error("device attribute: %s", cudaGetErrorString(e));
    return B200MOE_ERR_CUDA;
  }
  if (major != 10) {
    set_error("this library is built for sm_100a only; device %d has compute capability major %d", device, major);
    return B200MOE_ERR_UNSUPPORTED;
  }
  p->sms = sms;
  if (p->small) {
    p->bound = true;
    return B200MOE_OK;
  }
  int rc;
  if ((rc = configure_i8())) return rc;
  I8Gemm& g = p->gemm;
  const int pitch = int8_pitch(s.k);
  if ((rc = encode_i8(&g.tm_w, b->weight, s.n, s.k, pitch, 128, true))) return rc;
  if ((rc = encode_i8(&g.tm_act, b->x_q, s.tokens, s.k, pitch, p->token_tile, false))) return rc;
  g.w_scale = static_cast<const float*>(b->weight_scale);
  g.row_scale = static_cast<const float*>(b->x_scale);
  g.out = b->output;
  g.status = static_cast<int*>(b->status);
  g.groups = 1;
  g.rows = s.tokens;
  g.n_out = s.n;
  g.k = s.k;
  g.w_rows = s.n;
  g.token_tile = p->token_tile;
  g.boxes = p->boxes;
  g.split = p->split;
  int smem = 0;
  g.stages = i8_stages(2, g.boxes, g.token_tile, g.split, &smem);
  g.stream_weights = s.tokens <= p->token_tile;
  const long long items = static_cast<long long>((s.tokens + p->token_tile - 1) / p->token_tile) *
                          ((s.n + 128 * p->boxes - 1) / (128 * p->boxes));
  g.grid = static_cast<int>(p->split > 1 ? items * p->split : items < sms ? items : sms);
  p->bound = true;
  return B200MOE_OK;
}

int b200moe_linear_forward(B200MoeLinear* p, void* cuda_stream) {
  if (!p) {
    set_error("null argument");
    return B200MOE_ERR_INVALID;
  }
  if (!p->bound) {
    set_error("linear: no buffers bound; call b200moe_linear_bind first");
    return B200MOE_ERR_STATE;
  }
  if (p->shape.tokens == 0) return B200MOE_OK;
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  if (p->small) {
    const LinearSmall a{p->buf.x, p->shape.tokens > 1 ? p->buf.x_pitch : p->shape.k, static_cast<const int8_t*>(p->buf.weight),
                        static_cast<const float*>(p->buf.weight_scale), p->buf.output, static_cast<int8_t*>(p->buf.x_q),
                        static_cast<float*>(p->buf.x_scale), p->shape.dtype, p->shape.tokens, p->shape.k, p->shape.n, p->sms};
    const cudaError_t e = launch_linear_small(a, s);
    if (e != cudaSuccess) {
      set_error("linear launch: %s", cudaGetErrorString(e));
      return B200MOE_ERR_CUDA;
    }
    return B200MOE_OK;
  }
  QuantizeRows q{};
  q.x = p->buf.x;
  q.pitch = p->shape.tokens > 1 ? p->buf.x_pitch : p->shape.k;
  q.dtype = p->shape.dtype;
  q.rows = p->shape.tokens;
  q.k = p->shape.k;
  q.q = static_cast<int8_t*>(p->buf.x_q);
  q.scale = static_cast<float*>(p->buf.x_scale);
  cudaError_t e = launch_quantize_rows(q, s);
  if (e == cudaSuccess) e = launch_i8_product(p->gemm, p->shape.dtype, s);
  if (e != cudaSuccess) {
    set_error("linear launch: %s", cudaGetErrorString(e));
    return B200MOE_ERR_CUDA;
  }
  return B200MOE_OK;
}

void b200moe_linear_destroy(B200MoeLinear* p) { delete p; }

}  // extern "C"
