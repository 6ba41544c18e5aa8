// AdamW over many tensors in one launch, its states in fp32 or in 8 bits.
//
// Step t, every operation one correctly rounded fp32 operation, in this order:
//   m = m b1 + g (1 - b1),  v = v b2 + (g g)(1 - b2),  r = sqrt(v)
//   p = p (1 - lr wd) - (m (lr / (1 - b1^t))) / (r (1 / sqrt(1 - b2^t)) + eps)
// In 8 bits a block of 256 elements holds a = max|m|, s = max r and codes on quadratic grids, which keep 1 / 127^2 and
// 1 / 255^2 of the largest apart from zero:
//   c = sign(m) min(127, floor(sqrt(|m| (127^2 / a)) + z)) for m = c |c| (a (1 / 127^2))
//   u = min(255, floor(sqrt(r (255^2 / s)) + z)), 1 at least where r > 0, for r = u u (s (1 / 255^2))
// The second moment is held as r: what the step divides by, with half of v's range to cover, and no r > 0 is held as 0,
// so an element's step never grows because its r went below the grid.  z in [0, 1) runs through a Weyl sequence over
// steps and elements: a moment that moves by less than a code's distance in a step still moves on average, which with
// rounding to the nearest it would not (b2 = 0.999 moves r by 0.05% a step, neighbouring codes lie 0.8% apart at best).
// The average is right in the code, not in its square: with a root of n + f the value held is y + f (1 - f) on average, never
// too small, so a moment rises faster and falls slower by 1 / (2 n) of its way.  One that stays is held within 0.4% at n = 8
// and 0.03% from 18 on (simulated, b2 = 0.95 and 0.999).
// Blocks whose largest is below 2^-100 are held as zeros; one with an infinity or a NaN has scale NaN.  A finite gradient
// from 2^64 on has an infinite v: its element then only decays, in 32 bits for good; in 8 bits r is held as 2^63.
#include <cmath>

#include "train_ops.h"

namespace wfb {

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = WFB_ADAMW_BLOCK;          // elements of a block: a wave's 64 x 4
constexpr int kTileBlocks = 16;                  // blocks of one workgroup
constexpr float kLargestRoot = 0x1p63f;          // of a v past fp32's range, in 8 bits
constexpr int kMaxTensors = 64;                  // of one launch: the table travels with the kernel's arguments

struct Table {
  int n;
  uint32_t tile[kMaxTensors + 1];  // first workgroup of each tensor
  void* p[kMaxTensors];
  const void* g[kMaxTensors];
  int64_t len[kMaxTensors];
  int64_t first[kMaxTensors];  // of its elements in the state
};
static_assert(sizeof(Table) + sizeof(AdamWState) + sizeof(AdamWScalars) + 16 <= 4096, "kernel arguments");

// Four elements from any address that is a multiple of the element's size: gfx950 takes unaligned vectors.
struct __attribute__((packed, aligned(4))) F4 { float v[4]; };
struct __attribute__((packed, aligned(2))) H4 { uint16_t v[4]; };

template <int DT>
__device__ __forceinline__ void load4(const void* p, int64_t i, int n, float (&v)[4]) {
  if (n >= 4) {
    if constexpr (DT == WFB_F32) {
      const F4 x = *reinterpret_cast<const F4*>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = x.v[e];
    } else {
      const H4 x = *reinterpret_cast<const H4*>(reinterpret_cast<const uint16_t*>(p) + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = DT == WFB_BF16 ? bf16_bits_to_f32(x.v[e]) : f16_bits_to_f32(x.v[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < n ? load_elem<DT>(p, i + e) : 0.0f;
  }
}

template <int DT>
__device__ __forceinline__ void store4(void* p, int64_t i, int n, const float (&v)[4]) {
  if constexpr (DT == WFB_F32) {
    float* q = reinterpret_cast<float*>(p) + i;
    if (n >= 4) {
      F4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x.v[e] = v[e];
      *reinterpret_cast<F4*>(q) = x;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < n) q[e] = v[e];
    }
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(p) + i;
    H4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x.v[e] = DT == WFB_BF16 ? f32_to_bf16_rne(v[e]) : __builtin_bit_cast(uint16_t, (_Float16)v[e]);
    if (n >= 4) {
      *reinterpret_cast<H4*>(q) = x;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < n) q[e] = x.v[e];
    }
  }
}

// The largest of the wave's non-negative values; a NaN is the largest of all (its bits are).
__device__ __forceinline__ float wave_top(float v) {
  uint32_t u = __float_as_uint(v);
  auto up = [&](int o) { u = max(u, (uint32_t)o); };
  up(xor_lanes<1>((int)u));
  up(xor_lanes<2>((int)u));
  up(xor_lanes<4>((int)u));
  up(xor_lanes<8>((int)u));
  up(xor_lanes<16>((int)u));
  up(xor_lanes<32>((int)u));
  return __uint_as_float(u);
}

// Scale of a block whose largest is v.
__device__ __forceinline__ float scale_of(float v) {
  if (!(v <= 3.402823466e38f)) return __builtin_nanf("");
  return v < 7.888609052210118e-31f ? 0.0f : v;  // 2^-100
}

// The correctly rounded square root of x in [2^-100, 2^127]: x times the reciprocal root and one correction by the
// residual, whose fused rounding is the last.  Equal to the rounded double root for every significand under both
// parities of the exponent (all 2^24 tried on MI355X); five operations, where the compiler's sqrtf, which also
// takes subnormal numbers, needs about sixteen.
__device__ __forceinline__ float root_rn(float x) {
  const float y = __builtin_amdgcn_rsqf(x), s = __fmul_rn(x, y), h = 0.5f * y;
  return __builtin_fmaf(__builtin_fmaf(-s, s, x), h, s);
}

// sqrt of v >= 0, the few values between 0 and 2^-100 (and infinities and NaN) by sqrtf.
__device__ __forceinline__ float root_of(float v) {
  const bool plain = v >= 0x1p-100f && v <= 0x1p126f;
  float r = root_rn(plain ? v : 1.0f);
  if (__builtin_expect(!plain && v != 0.0f, 0)) return sqrtf(v);
  return plain ? r : 0.0f;
}

// n / d, correctly rounded: the reciprocal corrected once, the quotient once (every pair of significands tried on MI355X, 2^46)
// where no step leaves the normal numbers; the few others, an infinite or a zero divisor among them, by the compiler's
// division, about twice as long.
__device__ __forceinline__ float quotient(float n, float d) {
  const float a = fabsf(n);
  const bool plain = d >= 0x1p-40f && d <= 0x1p20f && a <= 0x1p80f && (a >= 0x1p-100f || a == 0.0f);
  if (__builtin_expect(!plain, 0)) return __fdiv_rn(n, d);
  float y = __builtin_amdgcn_rcpf(d);
  y = __builtin_fmaf(__builtin_fmaf(-d, y, 1.0f), y, y);
  const float q = __fmul_rn(n, y);
  return __builtin_fmaf(__builtin_fmaf(-d, q, n), y, q);
}

// Code of x >= 0 on the grid of `top` steps with k = top^2 / scale (below 2^-100 the root is next to nothing: 2^-50 there).
__device__ __forceinline__ int code_of(float x, float k, int top, float z) {
  return min((int)__fadd_rn(root_rn(fmaxf(__fmul_rn(x, k), 0x1p-100f)), z), top);
}

// A wave takes a block: its largest is a reduction over the lanes, and nothing is read twice.  fp32 states move 28 bytes an
// element (134M elements in six launches of up to 64 tensors 745-765 us, 4.9-5.05 TB/s), 8-bit states with bf16 gradients 14
// (139M elements 413 us, 4.7 TB/s; 476 with the compiler's sqrtf for an element's three roots; steps one behind the other).
template <int PDT, int GDT, int BITS>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Table tb, AdamWState st, AdamWScalars host,
                                                         const AdamWScalars* __restrict__ dev) {
  int k = 0;  // the tensor of this workgroup
  for (int step = kMaxTensors / 2; step; step /= 2)
    if (k + step < tb.n && tb.tile[k + step] <= blockIdx.x) k += step;
  const AdamWScalars c = dev ? *dev : host;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  void* const p = tb.p[k];
  const void* const g = tb.g[k];
  const int64_t len = tb.len[k], first = tb.first[k];
  const int64_t e0 = (int64_t)(blockIdx.x - tb.tile[k]) * (kTileBlocks * kBlock);
  for (int b = w; b < kTileBlocks; b += kThreads / 64) {
    const int64_t base = e0 + b * kBlock;
    if (base >= len) break;
    const int64_t i = base + 4 * lane, s = first + i;
    const int n = (int)min((int64_t)4, max((int64_t)0, len - i));
    float pv[4], gv[4], m[4], r[4];
    load4<PDT>(p, i, n, pv);
    load4<GDT>(g, i, n, gv);
    float v[4];
    if constexpr (BITS == 32) {
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(st.m) + s);
      const float4 y = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(st.v) + s);
      m[0] = x.x, m[1] = x.y, m[2] = x.z, m[3] = x.w;
      v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
    } else {
      const uint32_t mc = reinterpret_cast<const uint32_t*>(st.m)[s / 4], vc = reinterpret_cast<const uint32_t*>(st.v)[s / 4];
      const float ma = __fmul_rn(st.m_scale[s / kBlock], 1.0f / 16129.0f);
      const float va = __fmul_rn(st.v_scale[s / kBlock], 1.0f / 65025.0f);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float q = (float)(int8_t)(mc >> (8 * e)), u = (float)((vc >> (8 * e)) & 255u);
        m[e] = __fmul_rn(q * fabsf(q), ma);
        const float x = __fmul_rn(u * u, va);
        v[e] = __fmul_rn(x, x);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      m[e] = __fadd_rn(__fmul_rn(m[e], c.b1), __fmul_rn(gv[e], c.omb1));
      v[e] = __fadd_rn(__fmul_rn(v[e], c.b2), __fmul_rn(__fmul_rn(gv[e], gv[e]), c.omb2));
      if (e >= n) m[e] = v[e] = 0.0f;  // behind the tensor's end
      r[e] = root_of(v[e]);
      pv[e] = __fsub_rn(__fmul_rn(pv[e], c.decay),
                        quotient(__fmul_rn(m[e], c.rate), __fadd_rn(__fmul_rn(r[e], c.ib2), c.eps)));
    }
    store4<PDT>(p, i, n, pv);
    if constexpr (BITS == 32) {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(st.m) + s) = make_float4(m[0], m[1], m[2], m[3]);
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(st.v) + s) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      auto top4 = [](float a, float b, float c, float d) {  // (bits: a NaN is the largest)
        return __uint_as_float(max(max(__float_as_uint(fabsf(a)), __float_as_uint(fabsf(b))),
                                   max(__float_as_uint(fabsf(c)), __float_as_uint(fabsf(d)))));
      };
      const float a = scale_of(wave_top(top4(m[0], m[1], m[2], m[3])));
      float t = wave_top(top4(r[0], r[1], r[2], r[3]));
      if (__builtin_expect(t == __builtin_inff() && a == a, 0)) {  // (the wave agrees) a square past fp32, of a finite gradient
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = fminf(r[e], kLargestRoot);
        t = kLargestRoot;
      }
      t = scale_of(t);
      const float ka = a > 0.0f ? __fdiv_rn(16129.0f, a) : 0.0f, kt = t > 0.0f ? __fdiv_rn(65025.0f, t) : 0.0f;
      const uint32_t turn = (uint32_t)s * 0x9E3779B1u + c.turn;
      uint32_t q[4], u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z = (float)((turn + e * 0x9E3779B1u) >> 8) * 0x1p-24f;
        const int qa = code_of(fabsf(m[e]), ka, 127, z);
        q[e] = (uint32_t)(m[e] < 0.0f ? -qa : qa);
        u[e] = (uint32_t)max(code_of(r[e], kt, 255, z), r[e] > 0.0f ? 1 : 0);
      }
      auto pack = [](const uint32_t (&b)[4]) {  // the low bytes
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u),
                                     __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
      };
      // (no scale, no codes)
      reinterpret_cast<uint32_t*>(st.m)[s / 4] = a > 0.0f ? pack(q) : 0u;
      reinterpret_cast<uint32_t*>(st.v)[s / 4] = t > 0.0f ? pack(u) : 0u;
      if (lane == 0) {
        st.m_scale[s / kBlock] = a;
        st.v_scale[s / kBlock] = t;
      }
    }
  }
}

// The scalars of a step that is counted on the device, in double as the host computes them.
__global__ void adamw_scalars_kernel(double lr, const float* __restrict__ lr_dev, double b1, double b2, double wd,
                                     float eps, const int64_t* __restrict__ step_dev, AdamWScalars* __restrict__ out) {
  if (threadIdx.x) return;
  if (lr_dev) lr = (double)lr_dev[0];
  const int64_t t = step_dev[0];
  AdamWScalars c;
  c.b1 = (float)b1, c.omb1 = (float)(1.0 - b1), c.b2 = (float)b2, c.omb2 = (float)(1.0 - b2), c.eps = eps;
  c.decay = (float)(1.0 - lr * wd);
  c.rate = (float)(lr / (1.0 - pow(b1, (double)t)));
  c.ib2 = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
  c.turn = (uint32_t)t * 0x6A09E667u;
  *out = c;
}

// What the codes stand for, 4 elements a thread: 139M elements, 2 bytes read and 8 written each, 238 us (5.8 TB/s),
// 226 behind a step.
__global__ __launch_bounds__(kThreads) void adamw_values_kernel(AdamWState st, int64_t quads, float* __restrict__ m,
                                                                float* __restrict__ v) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < quads; i += (int64_t)gridDim.x * kThreads) {
    const uint32_t mc = reinterpret_cast<const uint32_t*>(st.m)[i], vc = reinterpret_cast<const uint32_t*>(st.v)[i];
    const float ma = __fmul_rn(st.m_scale[4 * i / kBlock], 1.0f / 16129.0f);
    const float va = __fmul_rn(st.v_scale[4 * i / kBlock], 1.0f / 65025.0f);
    float x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float q = (float)(int8_t)(mc >> (8 * e)), u = (float)((vc >> (8 * e)) & 255u);
      x[e] = __fmul_rn(q * fabsf(q), ma);
      const float r = __fmul_rn(u * u, va);
      y[e] = __fmul_rn(r, r);
    }
    reinterpret_cast<float4*>(m)[i] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(v)[i] = make_float4(y[0], y[1], y[2], y[3]);
  }
}

template <int PDT, int GDT>
void launch_bits(const Table& tb, unsigned grid, const AdamWState& st, const AdamWScalars& host, const AdamWScalars* dev,
                 hipStream_t s) {
  if (st.bits == 32)
    hipLaunchKernelGGL((adamw_kernel<PDT, GDT, 32>), dim3(grid), dim3(kThreads), 0, s, tb, st, host, dev);
  else
    hipLaunchKernelGGL((adamw_kernel<PDT, GDT, 8>), dim3(grid), dim3(kThreads), 0, s, tb, st, host, dev);
}

template <int PDT>
void launch_grad_type(const Table& tb, unsigned grid, int gdt, const AdamWState& st, const AdamWScalars& host,
                      const AdamWScalars* dev, hipStream_t s) {
  if (gdt == WFB_F32) launch_bits<PDT, WFB_F32>(tb, grid, st, host, dev, s);
  else if (gdt == WFB_BF16) launch_bits<PDT, WFB_BF16>(tb, grid, st, host, dev, s);
  else launch_bits<PDT, WFB_F16>(tb, grid, st, host, dev, s);
}

}  // namespace

hipError_t launch_adamw(const wfb_adamw_tensor* tensors, int64_t n, int pdt, int gdt, const AdamWState& st,
                        const AdamWScalars& host, const AdamWScalars* dev, hipStream_t s) {
  constexpr int64_t kTile = (int64_t)kTileBlocks * kBlock, kMostTiles = INT32_MAX / 2;
  Table tb;
  tb.n = 0;
  tb.tile[0] = 0;
  auto flush = [&]() -> hipError_t {
    if (tb.n == 0) return hipSuccess;
    const unsigned grid = tb.tile[tb.n];
    if (pdt == WFB_F32) launch_grad_type<WFB_F32>(tb, grid, gdt, st, host, dev, s);
    else if (pdt == WFB_BF16) launch_grad_type<WFB_BF16>(tb, grid, gdt, st, host, dev, s);
    else launch_grad_type<WFB_F16>(tb, grid, gdt, st, host, dev, s);
    tb.n = 0;
    return hipGetLastError();
  };
  int64_t next = 0;
  for (int64_t i = 0; i < n; ++i) {
    const int64_t first = next;
    next += (tensors[i].n + kBlock - 1) / kBlock * kBlock;
    if (tensors[i].n == 0 || !tensors[i].g) continue;
    const int64_t tiles = (tensors[i].n + kTile - 1) / kTile;
    if (tb.n == kMaxTensors || tb.tile[tb.n] + tiles > kMostTiles)
      if (const hipError_t e = flush(); e != hipSuccess) return e;
    tb.p[tb.n] = tensors[i].p;
    tb.g[tb.n] = tensors[i].g;
    tb.len[tb.n] = tensors[i].n;
    tb.first[tb.n] = first;
    tb.tile[tb.n + 1] = tb.tile[tb.n] + (uint32_t)tiles;
    ++tb.n;
  }
  return flush();
}

hipError_t launch_adamw_scalars(double lr, const float* lr_dev, double b1, double b2, double wd, float eps,
                                const int64_t* step_dev, AdamWScalars* out, hipStream_t s) {
  hipLaunchKernelGGL(adamw_scalars_kernel, dim3(1), dim3(64), 0, s, lr, lr_dev, b1, b2, wd, eps, step_dev, out);
  return hipGetLastError();
}

hipError_t launch_adamw_values(const AdamWState& st, int64_t elements, float* m, float* v, hipStream_t s) {
  const int64_t quads = elements / 4, groups = (quads + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(adamw_values_kernel, dim3((unsigned)(groups < 1 << 20 ? groups : 1 << 20)), dim3(kThreads), 0, s,
                     st, quads, m, v);
  return hipGetLastError();
}

}  // namespace wfb
