// The gated feed-forward product of two ternary projections of the same activations, and its backward pass.
//
//   [gate | up] = (codes t^T) a w,   h = act(gate) up
//   d_gate = gh up act'(gate),  d_up = gh act(gate)
//   grad_x = [d_gate w_gate | d_up w_up] t,   grad_W = [d_gate | d_up]^T (codes a)      (straight through both quantisers)
// silu(g) = g s, silu'(g) = s + g s (1 - s), s = 1 / (1 + exp(-g));  relu2(g) = max(g, 0)^2, its slope 2 max(g, 0).
// The float module that this trains is WF/models/ffn.py:10-45 over WF/models/bitlinear.py:86-113.
#include "train_ops.h"

namespace wfb {

namespace {

template <int ACT>
__device__ __forceinline__ void act_and_slope(float g, float& act, float& slope) {
  if constexpr (ACT == WFB_ACT_SILU) {
    const float s = __fdiv_rn(1.0f, 1.0f + exp2_fixed(-g * 1.4426950408889634f));
    act = g * s;
    slope = s + g * s * (1.0f - s);
  } else {
    const float r = fmaxf(g, 0.0f);
    act = r * r;
    slope = 2.0f * r;
  }
}

__device__ __forceinline__ void store_as(void* o, int dt, int64_t i, float y) {
  if (dt == WFB_F32) reinterpret_cast<float*>(o)[i] = y;
  else if (dt == WFB_BF16) reinterpret_cast<uint16_t*>(o)[i] = f32_to_bf16_rne(y);
  else reinterpret_cast<uint16_t*>(o)[i] = __builtin_bit_cast(uint16_t, (_Float16)y);
}

template <int ACT>
__global__ __launch_bounds__(256) void gated_kernel(const float* __restrict__ gu, int64_t m, int64_t f,
                                                    void* __restrict__ h, int h_dtype) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= m * f) return;
  const int64_t row = i / f, col = i - row * f;
  store_as(h, h_dtype, i, glu<ACT>(gu[row * 2 * f + col], gu[row * 2 * f + f + col]));
}

template <int ACT, int GDT>
__global__ __launch_bounds__(256) void gated_grad_kernel(const float* __restrict__ gu, const void* __restrict__ gh,
                                                         int64_t ldg, int64_t m, int64_t f,
                                                         const float* __restrict__ scales, float* __restrict__ d,
                                                         float* __restrict__ ds, float* __restrict__ one) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i == 0) one[0] = 1.0f;
  if (i >= m * f) return;
  const int64_t row = i / f, col = i - row * f, o = row * 2 * f + col;
  const float gate = gu[o], up = gu[o + f], g = load_elem<GDT>(gh, row * ldg + col);
  float act, slope;
  act_and_slope<ACT>(gate, act, slope);
  const float dg = g * up * slope, du = g * act;
  d[o] = dg, d[o + f] = du;
  ds[o] = dg * scales[0], ds[o + f] = du * scales[1];
}

constexpr int64_t align256(int64_t b) { return (b + 255) / 256 * 256; }

}  // namespace

int64_t gated_workspace_floats(int64_t m, int64_t f, int64_t k) { return m * 2 * f; }

hipError_t launch_gated(const GatedForward& p, hipStream_t s) {
  for (int i = 0; i < 2; ++i) {
    Epilogue e{};
    e.nseg = 1;
    e.a_scale = p.a_scale;
    e.ws_dev = p.scales + i;
    e.out = p.gate_up + i * p.f;
    e.out_dtype = WFB_F32;
    e.ldo = 2 * p.f;
    const uint8_t* w = p.qw + i * p.f * (p.k / 4);
    const bool gemv = p.m <= 2 && p.k <= 32768 && p.f * (p.k / 4) <= INT32_MAX && (p.m - 1) * p.lda + p.k <= INT32_MAX;
    const hipError_t st = gemv ? launch_gemv_i2s(w, (int)p.f, (int)p.k, p.codes, (int)p.m, p.lda, e, s)
                               : launch_gemm_i2s(w, (int)p.f, (int)p.k, p.codes, (int)p.m, p.lda, e, s);
    if (st != hipSuccess) return st;
  }
  const unsigned grid = (unsigned)((p.m * p.f + 255) / 256);
  if (p.act == WFB_ACT_SILU)
    hipLaunchKernelGGL(gated_kernel<WFB_ACT_SILU>, dim3(grid), dim3(256), 0, s, p.gate_up, p.m, p.f, p.h, p.h_dtype);
  else
    hipLaunchKernelGGL(gated_kernel<WFB_ACT_RELU2>, dim3(grid), dim3(256), 0, s, p.gate_up, p.m, p.f, p.h, p.h_dtype);
  return hipGetLastError();
}

int64_t gated_grad_workspace(const GatedGrad& p) {
  const int64_t d = align256(4 * p.m * 2 * p.f);
  const int64_t x = p.gx ? grad_x_workspace(p.m, 2 * p.f, p.k, WFB_F32) : 0;
  const int64_t w = p.gw ? grad_w_workspace(p.m, 2 * p.f, p.k) : 0;
  return 256 + 2 * d + (x > w ? x : w);
}

hipError_t launch_gated_grad(const GatedGrad& p, void* work, hipStream_t s) {
  const int64_t size = align256(4 * p.m * 2 * p.f);
  char* ws = static_cast<char*>(work);
  float* one = reinterpret_cast<float*>(ws);
  float* d = reinterpret_cast<float*>(ws + 256);
  float* ds = reinterpret_cast<float*>(ws + 256 + size);
  void* rest = ws + 256 + 2 * size;
  const unsigned grid = (unsigned)((p.m * p.f + 255) / 256);
#define WFB_GG(ACT, DT) \
  hipLaunchKernelGGL((gated_grad_kernel<ACT, DT>), dim3(grid), dim3(256), 0, s, p.gate_up, p.gh, p.ldg, p.m, p.f, \
                     p.scales, d, ds, one)
#define WFB_GGD(ACT)                                     \
  do {                                                   \
    if (p.gh_dtype == WFB_F32) WFB_GG(ACT, WFB_F32);     \
    else if (p.gh_dtype == WFB_BF16) WFB_GG(ACT, WFB_BF16); \
    else WFB_GG(ACT, WFB_F16);                           \
  } while (0)
  if (p.act == WFB_ACT_SILU) WFB_GGD(WFB_ACT_SILU);
  else WFB_GGD(WFB_ACT_RELU2);
#undef WFB_GGD
#undef WFB_GG
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.gx)
    e = launch_grad_x(ds, WFB_F32, 2 * p.f, p.m, 2 * p.f, p.qw, p.k, p.k_pad, one, p.gx, p.gx_dtype, p.k, rest, s);
  if (e == hipSuccess && p.gw)
    e = launch_grad_w(d, WFB_F32, 2 * p.f, p.m, 2 * p.f, p.codes, p.lda, p.a_scale, p.k, p.gw, p.gw_dtype, p.k, nullptr,
                      0, rest, s);
  return e;
}

}  // namespace wfb
