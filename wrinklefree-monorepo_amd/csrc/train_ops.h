// Launchers of the training-step operators: the gated product's forward and backward pass (gated.hip), the norm of query
// and key heads with the rotary embedding (qk_rope.hip), AdamW over many tensors (adamw.hip).
#pragma once

#include "wfb_common.h"

namespace wfb {

// One of the two sides (queries, keys) of the rotation: x [batch, t, heads, head_dim], strides in elements.
struct HeadRows {
  const void* x;
  int64_t xb, xt, xh;
  const void* g;  // gradient at the output (backward only)
  int64_t gb, gt, gh;
  const void* w;  // norm weight [head_dim], or null: no norm
  int wdt;
  void* out;  // contiguous: the output, or the gradient of x (may be null in the backward pass)
  int heads;
};

struct QkRope {
  HeadRows side[2];
  const float* cos;
  const float* sin;
  int64_t rope_len;
  int rotary;       // elements turned, R <= head_dim
  int interleaved;  // pairs (2i, 2i + 1) instead of (i, i + R / 2)
  const void* pos;  // int32 / int64, or null: start + t
  int pos64;
  int64_t pb, pt;
  int64_t start;
  int64_t batch, t;
  int head_dim;
  float eps;
};

// Groups of heads that one group of lanes takes; the kernels count them in 32 bits (below 2^31).
int64_t qk_tasks(const QkRope& p);
// Workgroups of the backward pass, each of which leaves one row [2][head_dim] of partial weight gradients.
int qk_grad_parts(const QkRope& p);
hipError_t launch_qk_rope(const QkRope& p, int dtype, hipStream_t s);
// gw: [2][head_dim] fp32 sums in `work` (qk_grad_parts rows), rounded into gw0 / gw1 of gdt0 / gdt1 (null: not wanted)
hipError_t launch_qk_rope_grad(const QkRope& p, int dtype, void* gw0, int gdt0, void* gw1, int gdt1, float* work,
                               hipStream_t s);

// What a step's arithmetic takes, each rounded to fp32; on the host or, for steps counted on the device, in memory.
struct AdamWScalars {
  float b1, omb1, b2, omb2, eps, decay, rate, ib2;
  uint32_t turn;  // step * 0x6A09E667
};

struct AdamWState {
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  int bits;
};

hipError_t launch_adamw(const wfb_adamw_tensor* tensors, int64_t n, int pdt, int gdt, const AdamWState& st,
                        const AdamWScalars& host, const AdamWScalars* dev, hipStream_t s);
hipError_t launch_adamw_scalars(double lr, const float* lr_dev, double b1, double b2, double wd, float eps,
                                const int64_t* step_dev, AdamWScalars* out, hipStream_t s);
hipError_t launch_adamw_values(const AdamWState& st, int64_t elements, float* m, float* v, hipStream_t s);

// h [m, f] = act(gate) * up of the gate|up product of int8 codes; gate_up takes both products, or is null.
struct GatedForward {
  const uint8_t* qw;  // [2f, k / 4]
  int64_t f, k;
  const int8_t* codes;
  int64_t m, lda;
  const float* a_scale;
  const float* scales;  // [2]
  int act;
  void* h;
  int h_dtype;
  float* gate_up;
};
hipError_t launch_gated(const GatedForward& p, hipStream_t s);

struct GatedGrad {
  const float* gate_up;
  const void* gh;  // [m, f]
  int gh_dtype;
  int64_t ldg, m, f;
  int act;
  const uint8_t* qw;  // [2f, k_pad / 4]
  int64_t k, k_pad;
  const float* scales;
  const int8_t* codes;
  int64_t lda;
  const float* a_scale;
  void* gx;  // [m, k] or null
  int gx_dtype;
  void* gw;  // [2f, k] or null
  int gw_dtype;
  bool wide_x, wide_w;  // operands in two planes for a bf16 result too
};
int64_t gated_grad_workspace(const GatedGrad& p);
hipError_t launch_gated_grad(const GatedGrad& p, void* work, hipStream_t s);

}  // namespace wfb
