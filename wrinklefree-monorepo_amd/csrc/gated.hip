// The gated feed-forward product of two ternary projections of the same activations, and its backward pass.
//
//   [gate | up] = (codes t^T) a w,   h = act(gate) up
//   d_gate = gh up act'(gate),  d_up = gh act(gate)
//   grad_x = [d_gate w_gate | d_up w_up] t,   grad_W = [d_gate | d_up]^T (codes a)      (straight through both quantisers)
// silu(g) = g s, silu'(g) = s + g s (1 - s), s = 1 / (1 + exp(-g));  relu2(g) = max(g, 0)^2, its slope 2 max(g, 0).
// The float module that this trains is WF/models/ffn.py:10-45 over WF/models/bitlinear.py:86-113.
//
// The backward pass.  Both products have one operand that fp16 holds exactly (t, the int8 codes).  The other, d times a
// scale, enters as one or two fp16 planes of d 2^e, e chosen for each row of the product's left operand so that the row's
// largest lies in [2^14, 2^15): a plane holds 11 bits of a value down to 2^-28 of the largest, two hold 22 down to
// 2^-18 (below, an error of 2^-40 of the largest).  One plane where the result is bf16 (8 bits: each term is then off by
// an eighth of what a bf16 gradient of the projections would be, and the result's error against 64 bits grows by less than 1%)
// unless the caller asks for two; two for fp32 results, and for fp16 ones, whose own half step one plane's error of a term equals
// (2000 x 4096 x 14336 in bf16 1385 us, in bf16 with two planes 2005, in fp16 1990; 4096 x 2560 x 6912 in bf16 with fp32
// weights, whose gradient takes two anyway, 1110 and 1320).  Against three bf16 planes, which need no e, that is a
// third and two thirds of the products.  Sums are fp32; the result times 2^-e is rounded once.
// An infinity or a NaN in a row of d leaves that row of the result without finite values worth the name, and no other.
//
// Three passes: the largest of every row and column of d (gated_top_kernel, gated_scale_kernel), the planes in the order in
// which the products read them (gated_planes_kernel; ternary weights and codes likewise), the two products (grad_tile.h).
// The largest values have to be known before the first plane is written, so d is formed twice, and both passes are bound by
// memory: 4096 tokens of 2560 -> 6912 with fp32 weights 73 us (393 MB with the transposed operands), 6 for the factors and
// 120 us (622 MB, 5.2 TB/s).  The products take 440 (two planes) and 259 us there, 1.32 and 1.12 PFLOP/s.
#include <algorithm>

#include "grad_tile.h"
#include "train_ops.h"

namespace wfb {

namespace {

constexpr int64_t gated_pad(int64_t f) { return (f + 63) / 64 * 64; }  // columns of one product in gate_up

// ---- backward: what the layout kernels share -------------------------------------------------------

struct GradSrc {
  const float* gu;  // [m][2 fp]
  const void* gh;
  int64_t ldg;
  bool vec;  // gh's groups of 4 columns start at multiples of 4 elements
  int m, f, fp;
  const float* scales;   // [2]
  const float* a_scale;  // [m]
};

// (d_gate, d_up).  exp(-gate) by the hardware's base-2 exponential of the rounded product and a correction for what the
// product's rounding left (|gate| 2^-24 of the result): four roundings whatever the gate.  1 - s as exp(-gate) s, which keeps its
// digits where s is next to 1.  Nine operations more an element than without, which the passes over memory hide (2000 x 14336:
// the whole step 1344 us both).
template <int ACT>
__device__ __forceinline__ void gated_slopes(float gate, float up, float g, float& dg, float& du) {
  if constexpr (ACT == WFB_ACT_SILU) {
    constexpr float kHi = -1.4426950408889634f, kLo = (float)(-1.4426950408889634 - (double)kHi);  // -1 / ln 2
    // (within [-88, 120] exp(-gate) is finite and the correction small; below, s and what it multiplies are next to nothing,
    // above, s is 1; a NaN stays one in a)
    const float low = gate < -88.0f ? -88.0f : gate, e = fminf(low, 120.0f);
    const float p = e * kHi, rest = __builtin_fmaf(e, kLo, __builtin_fmaf(e, kHi, -p));
    const float t = __builtin_amdgcn_exp2f(p), x = __builtin_fmaf(t, rest * 0.6931471805599453f, t);
    const float s = __builtin_amdgcn_rcpf(1.0f + x), a = low * s;
    dg = g * up * __builtin_fmaf(a, x * s, s);
    du = g * a;
  } else {
    const float r = fmaxf(gate, 0.0f);
    dg = g * up * (2.0f * r);
    du = g * (r * r);
  }
}

// d of columns c .. c + 3 of row `row` (both clamped into range; columns past f give 0).
template <int ACT, int GDT>
__device__ __forceinline__ void load_d(const GradSrc& p, int row, int c, float (&dg)[4], float (&du)[4]) {
  const float* gu = p.gu + (int64_t)row * 2 * p.fp + c;
  const float4 gt = *reinterpret_cast<const float4*>(gu), ut = *reinterpret_cast<const float4*>(gu + p.fp);
  const float gate[4] = {gt.x, gt.y, gt.z, gt.w}, up[4] = {ut.x, ut.y, ut.z, ut.w};
  float g[4];
  const int64_t at = row * p.ldg + c;
  if (p.vec && c + 4 <= p.f) {
    if constexpr (GDT == WFB_F32) {
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.gh) + at);
      g[0] = x.x, g[1] = x.y, g[2] = x.z, g[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p.gh) + at);
      const uint32_t w[2] = {x.x, x.y};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint16_t b = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
        g[e] = GDT == WFB_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] = load_elem<GDT>(p.gh, at - c + min(c + e, p.f - 1));
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    gated_slopes<ACT>(gate[e], up[e], g[e], dg[e], du[e]);
    if (c + e >= p.f) dg[e] = du[e] = 0.0f;
  }
}

__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The largest magnitude (as bits: a NaN is the largest) of every row of [d_gate w_gate | d_up w_up] and of every
// column of d a, over tiles of 64 columns and `rows` rows: row_part[f tile][m], col_part[row tile][2 f].
template <int ACT, int GDT>
__device__ __forceinline__ void gated_top(const GradSrc& p, int bx, int by, int rows, uint32_t* __restrict__ row_part,
                                          uint32_t* __restrict__ col_part, uint32_t (&red)[2][16][64]) {
  const int cq = threadIdx.x & 15, r0 = threadIdx.x >> 4, c = bx * 64 + 4 * cq, m0 = by * rows;
  const float w0 = p.scales[0], w1 = p.scales[1];
  uint32_t cg[4] = {0, 0, 0, 0}, cu[4] = {0, 0, 0, 0};
  for (int j0 = 0; j0 < rows; j0 += 64) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = m0 + j0 + r0 + 16 * j, rc = min(row, p.m - 1);
      float dg[4], du[4];
      load_d<ACT, GDT>(p, rc, c, dg, du);
      const float a = p.a_scale[rc];
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        top = max(top, max(mag(dg[e] * w0), mag(du[e] * w1)));
        cg[e] = max(cg[e], mag(dg[e] * a));
        cu[e] = max(cu[e], mag(du[e] * a));
      }
      top = max(top, (uint32_t)xor_lanes<1>((int)top));
      top = max(top, (uint32_t)xor_lanes<2>((int)top));
      top = max(top, (uint32_t)xor_lanes<4>((int)top));
      top = max(top, (uint32_t)xor_lanes<8>((int)top));
      if (cq == 0 && row < p.m) row_part[(int64_t)bx * p.m + row] = top;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) red[0][r0][4 * cq + e] = cg[e], red[1][r0][4 * cq + e] = cu[e];
  __syncthreads();
  if (threadIdx.x < 128) {
    const int half = threadIdx.x >> 6, i = threadIdx.x & 63, f = bx * 64 + i;
    uint32_t v = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) v = max(v, red[half][k][i]);
    if (f < p.f) col_part[(int64_t)by * 2 * p.f + half * p.f + f] = v;
  }
}

// I2_S codes of the 2f weight rows as fp16 {-1, 0, 1}, dst[k][2 fp]: row n of gate in column n, of up in column fp + n,
// zeros between.  One 128-weight block of 64 rows per workgroup.
__device__ __forceinline__ void gated_weights_t(const uint8_t* __restrict__ qw, int64_t row_bytes, int f, int fp, int K,
                                                int bx, int b, uint16_t* __restrict__ dst, uint8_t (&tile)[64][36]) {
  const int n0 = bx * 64;  // columns n0 .. n0 + 63 of dst lie in one half (fp % 64 == 0)
  const int up = n0 >= fp, first = up ? n0 - fp : n0;
  {
    const int r = threadIdx.x >> 2, c8 = threadIdx.x & 3;  // 8 bytes of one row per thread
    const int n = first + r;
    const uint2 w = *reinterpret_cast<const uint2*>(qw + (int64_t)(up * f + min(n, f - 1)) * row_bytes + 32 * b + 8 * c8);
    uint32_t* t = reinterpret_cast<uint32_t*>(&tile[r][8 * c8]);  // (code 1 = weight 0)
    t[0] = n < f ? w.x : 0x55555555u;
    t[1] = n < f ? w.y : 0x55555555u;
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int idx = threadIdx.x + 256 * it, ch = idx & 7, kl = idx >> 3;  // 8 rows n of column kl
    const int k = 128 * b + kl;
    if (k >= K) continue;
    const int j = kl & 31, sh = 6 - 2 * (kl >> 5);
    union { uint16_t h[8]; uint4 q; } o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int code = (tile[8 * ch + e][j] >> sh) & 3;
      o.h[e] = code == 0 ? 0xbc00u : code == 1 ? 0u : 0x3c00u;  // -1, 0, 1 in fp16
    }
    *reinterpret_cast<uint4*>(dst + (int64_t)k * 2 * fp + n0 + 8 * ch) = o.q;
  }
}

// The first launch of the backward pass: the largest of d's rows and columns, and the operands that do not wait for
// them, the transposed weights (columns x 64 by blocks of 128) and codes (tokens x 64 by columns x 64).
struct Operands {
  const uint8_t* qw;
  int64_t row_bytes;
  const int8_t* codes;
  int64_t lda;
  bool vec;  // codes' rows 16-byte aligned
  int K, mp;
  uint16_t *wt, *ct;  // null: not wanted
  int top_rows, tops, top_tiles, weights, weight_tiles, code_tiles;  // workgroups of each part, tiles of its first dimension
};

template <int ACT, int GDT>
__global__ __launch_bounds__(256) void gated_top_kernel(GradSrc p, Operands o, uint32_t* __restrict__ row_part,
                                                        uint32_t* __restrict__ col_part) {
  __shared__ union {
    uint32_t red[2][16][64];
    __attribute__((aligned(4))) uint8_t w[64][36];
    __attribute__((aligned(4))) int8_t c[64][68];
  } lds;
  int b = blockIdx.x;
  if (b < o.tops) return gated_top<ACT, GDT>(p, b % o.top_tiles, b / o.top_tiles, o.top_rows, row_part, col_part, lds.red);
  b -= o.tops;
  if (b < o.weights)
    return gated_weights_t(o.qw, o.row_bytes, p.f, p.fp, o.K, b % o.weight_tiles, b / o.weight_tiles, o.wt, lds.w);
  b -= o.weights;
  const int m0 = b % o.code_tiles, k0 = b / o.code_tiles;
  if (o.vec) codes_t<true, true>(o.codes, o.lda, p.m, o.K, o.mp, m0, k0, o.ct, lds.c);
  else codes_t<false, true>(o.codes, o.lda, p.m, o.K, o.mp, m0, k0, o.ct, lds.c);
}

// What a row whose largest is `top` is multiplied by: the power of two that brings it into [2^14, 2^15), 2^126 at most; 1
// where there is none (zero, infinity, NaN).
__device__ __forceinline__ float plane_scale(uint32_t top) {
  const int e = (int)(top >> 23);
  if (top == 0 || e == 255) return 1.0f;
  return __uint_as_float((uint32_t)min(268 - max(e, 1), 253) << 23);  // 2^(141 - e), biased: 141 - e + 127
}

// The factors of rows and columns and their inverses: scale[0 .. n), inverse[0 .. n), rows first.
__global__ __launch_bounds__(256) void gated_scale_kernel(const uint32_t* __restrict__ row_part, int row_tiles, int m,
                                                          const uint32_t* __restrict__ col_part, int col_tiles, int n,
                                                          float* __restrict__ scale, float* __restrict__ inverse) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= m + n) return;
  const uint32_t* src = i < m ? row_part + i : col_part + (i - m);
  const int tiles = i < m ? row_tiles : col_tiles, ld = i < m ? m : n;
  uint32_t v = 0;
  for (int t = 0; t < tiles; t += 32) {  // (the last one again past the end: 32 loads in flight, of one thread's chain)
#pragma unroll
    for (int u = 0; u < 32; ++u) v = max(v, src[(int64_t)min(t + u, tiles - 1) * ld]);
  }
  const float s = plane_scale(v);
  scale[i] = s;
  inverse[i] = 1.0f / s;  // (a power of two)
}

// Planes of a scaled value: the nearest fp16, and the nearest of what is left.
template <int P>
__device__ __forceinline__ void split_f16(float v, uint16_t (&h)[2]) {
  const _Float16 a = (_Float16)v;
  h[0] = __builtin_bit_cast(uint16_t, a);
  if constexpr (P == 2) {
    const float r = v - (float)a;
    h[1] = mag(v) < 0x7f800000u ? __builtin_bit_cast(uint16_t, (_Float16)r) : (uint16_t)0;
  }
}

// Both operands' planes from one reading of d, a 64 x 64 tile of each half per workgroup: px[plane][m][2 fp] of d w 2^e as
// it lies, pw[plane][2 f][mp] of d a 2^e through LDS (rows of 65 words: either side of the transpose without bank
// conflicts).  Columns f .. fp and tokens m .. mp are zeros.
template <int ACT, int GDT, int PX, int PW>
__global__ __launch_bounds__(256) void gated_planes_kernel(GradSrc p, const float* __restrict__ row_scale,
                                                           const float* __restrict__ col_scale, int mp,
                                                           uint16_t* __restrict__ px, uint16_t* __restrict__ pw) {
  __shared__ float tile[PW ? 2 : 1][PW ? 64 : 1][65];
  const int cq = threadIdx.x & 15, r0 = threadIdx.x >> 4, f0 = blockIdx.x * 64, c = f0 + 4 * cq, m0 = blockIdx.y * 64;
  const float w0 = p.scales[0], w1 = p.scales[1];
  float sg[4], su[4];
  if constexpr (PW > 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int f = min(c + e, p.f - 1);
      sg[e] = col_scale[f], su[e] = col_scale[p.f + f];
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = m0 + r0 + 16 * j, rc = min(row, p.m - 1);
    float dg[4], du[4];
    load_d<ACT, GDT>(p, rc, c, dg, du);
    if constexpr (PX > 0) {
      const float s = row_scale[rc];
      union { uint16_t h[4]; uint2 q; } og[2], ou[2];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint16_t hg[2], hu[2];
        split_f16<PX>(dg[e] * w0 * s, hg);
        split_f16<PX>(du[e] * w1 * s, hu);
#pragma unroll
        for (int q = 0; q < PX; ++q) og[q].h[e] = hg[q], ou[q].h[e] = hu[q];
      }
      if (row < p.m) {
#pragma unroll
        for (int q = 0; q < PX; ++q) {
          uint16_t* o = px + ((int64_t)q * p.m + row) * 2 * p.fp + c;
          *reinterpret_cast<uint2*>(o) = og[q].q;
          *reinterpret_cast<uint2*>(o + p.fp) = ou[q].q;
        }
      }
    }
    if constexpr (PW > 0) {
      const float a = p.a_scale[rc];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        tile[0][r0 + 16 * j][4 * cq + e] = row < p.m ? dg[e] * a * sg[e] : 0.0f;
        tile[1][r0 + 16 * j][4 * cq + e] = row < p.m ? du[e] * a * su[e] : 0.0f;
      }
    }
  }
  if constexpr (PW > 0) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int idx = threadIdx.x + 256 * j, ch = idx & 7, fl = (idx >> 3) & 63, half = idx >> 9;
      if (f0 + fl >= p.f) continue;
      union { uint16_t h[8]; uint4 q; } o[2];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint16_t h[2];
        split_f16<PW>(tile[half][8 * ch + e][fl], h);
#pragma unroll
        for (int q = 0; q < PW; ++q) o[q].h[e] = h[q];
      }
#pragma unroll
      for (int q = 0; q < PW; ++q)
        *reinterpret_cast<uint4*>(pw + ((int64_t)q * 2 * p.f + half * p.f + f0 + fl) * mp + m0 + 8 * ch) = o[q].q;
    }
  }
}

// Fitted to the times of every form, every split of all tiles and of the tiles past the last full round, of 28 shapes from
// 16 x 2560 x 13824 to 28672 x 4096 x 2048 with one and two planes: the picks take 1.03 times the fastest on average, 1.24
// at most (36 against 29 us).
constexpr Variant kVariants16[] = {{1, 256, 256, 32, 1, 1.45, 12.4, 0.8}, {1, 128, 256, 64, 1, 1.44, 8.8, 0.85},
                                   {1, 128, 128, 64, 2, 1.12, 7.9},       {1, 64, 128, 64, 3, 0.82, 4},
                                   {2, 256, 256, 32, 1, 1.57, 10.6, 0.8}, {2, 128, 256, 32, 2, 1.29, 8.6},
                                   {2, 64, 128, 32, 4, 0.92, 2.4}};
constexpr int kNumVariants16 = sizeof(kVariants16) / sizeof(kVariants16[0]);

Plan plan16(int planes, int64_t I, int64_t J, int64_t C) { return plan_of(kVariants16, kNumVariants16, planes, I, J, C, 0.32); }

hipError_t run_gemm16(GradGemm p, const Plan& pl, int64_t C, float* parts, hipStream_t s) {
  set_plan(p, pl, kVariants16, C, parts);
  switch (pl.variant) {  // kVariants16
    case 0: return launch_tiles<true, 1, 4, 2, 2, 4, 32, 2, 4>(p, pl, s);
    case 1: return launch_tiles<true, 1, 2, 4, 2, 2, 64, 1, 3>(p, pl, s);
    case 2: return launch_tiles<true, 1, 2, 2, 2, 2, 64, 2>(p, pl, s);
    case 3: return launch_tiles<true, 1, 1, 2, 2, 2, 64, 3>(p, pl, s);
    case 4: return launch_tiles<true, 2, 4, 2, 2, 4, 32, 2, 3>(p, pl, s);
    case 5: return launch_tiles<true, 2, 2, 4, 2, 2, 32, 2>(p, pl, s);
    default: return launch_tiles<true, 2, 1, 2, 2, 2, 32, 4>(p, pl, s);
  }
}

// The backward pass's buffers, one behind the other in its workspace.
struct GradLayout {
  int px, pw;  // planes, 0: result not wanted
  int64_t fp, mp, top_rows, row_tiles, col_tiles;
  int64_t row_part, col_part, scale, inverse, ax, bx, aw, bw, parts_x, parts_w, bytes;
  Plan plan_x, plan_w;
};

GradLayout grad_layout(const GatedGrad& p) {
  GradLayout l{};
  l.px = !p.gx ? 0 : p.gx_dtype == WFB_BF16 && !p.wide_x ? 1 : 2;
  l.pw = !p.gw ? 0 : p.gw_dtype == WFB_BF16 && !p.wide_w ? 1 : 2;
  l.fp = gated_pad(p.f);
  l.mp = pad_to(p.m, kPad);
  l.row_tiles = l.fp / 64;
  // Rows of a tile that gated_top takes: 256, or 64 where that makes fewer than three workgroups a CU (509 x 1536 6.2 against
  // 13.9 us, 1024 x 6912 27 against 35, 700 x 14336 62 against 74; 2048 x 6912 44 both, 2000 x 14336 102 against 99).  Many
  // rows leave enough of them, and more parts would only lengthen the columns' maxima.
  l.top_rows = p.m <= 4096 && l.row_tiles * ((p.m + 255) / 256) < 768 ? 64 : 256;
  l.col_tiles = (p.m + l.top_rows - 1) / l.top_rows;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += align256(bytes);
    return o;
  };
  l.row_part = take(4 * l.row_tiles * p.m);
  l.col_part = take(4 * l.col_tiles * 2 * p.f);
  l.scale = take(4 * (p.m + 2 * p.f));
  l.inverse = take(4 * (p.m + 2 * p.f));
  if (l.px) {
    l.plan_x = plan16(l.px, p.m, p.k, 2 * l.fp);
    l.ax = take(2 * l.px * p.m * 2 * l.fp);
    l.bx = take(2 * p.k * 2 * l.fp);
    l.parts_x = take(part_bytes_of(kVariants16, l.plan_x));
  }
  if (l.pw) {
    l.plan_w = plan16(l.pw, 2 * p.f, p.k, p.m);
    l.aw = take(2 * l.pw * 2 * p.f * l.mp);
    l.bw = take(2 * p.k * l.mp);
    l.parts_w = take(part_bytes_of(kVariants16, l.plan_w));
  }
  l.bytes = at;
  return l;
}

template <int ACT, int GDT>
hipError_t launch_layouts(const GradSrc& src, const Operands& ops, const GradLayout& l, char* ws, hipStream_t s) {
  auto* row_part = reinterpret_cast<uint32_t*>(ws + l.row_part);
  auto* col_part = reinterpret_cast<uint32_t*>(ws + l.col_part);
  auto* scale = reinterpret_cast<float*>(ws + l.scale);
  auto* inverse = reinterpret_cast<float*>(ws + l.inverse);
  const int grid0 = ops.tops + ops.weights + (ops.ct ? ops.code_tiles * ((ops.K + 63) / 64) : 0);
  hipLaunchKernelGGL((gated_top_kernel<ACT, GDT>), dim3(grid0), dim3(256), 0, s, src, ops, row_part, col_part);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int n = src.m + 2 * src.f;
  hipLaunchKernelGGL(gated_scale_kernel, dim3((n + 255) / 256), dim3(256), 0, s, row_part, (int)l.row_tiles, src.m, col_part,
                     (int)l.col_tiles, 2 * src.f, scale, inverse);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const dim3 grid((unsigned)(l.fp / 64), (unsigned)(l.mp / 64));
  auto* ax = reinterpret_cast<uint16_t*>(ws + l.ax);
  auto* aw = reinterpret_cast<uint16_t*>(ws + l.aw);
#define WFB_PLANES(PX, PW)                                                                                           \
  hipLaunchKernelGGL((gated_planes_kernel<ACT, GDT, PX, PW>), grid, dim3(256), 0, s, src, scale, scale + src.m, (int)l.mp, \
                     ax, aw)
  switch (3 * l.px + l.pw) {
    case 1: WFB_PLANES(0, 1); break;
    case 2: WFB_PLANES(0, 2); break;
    case 3: WFB_PLANES(1, 0); break;
    case 4: WFB_PLANES(1, 1); break;
    case 5: WFB_PLANES(1, 2); break;
    case 6: WFB_PLANES(2, 0); break;
    case 7: WFB_PLANES(2, 1); break;
    default: WFB_PLANES(2, 2); break;
  }
#undef WFB_PLANES
  return hipGetLastError();
}

}  // namespace

// Up to 32 tokens whose products nobody keeps take the decode kernels' gated epilogue, all else pair tiles (2560 x 6912: 8
// tokens 7.3 against 11.1 us, 32 10.1 against 12.9, 48 14.1 against 13.1; 4096 x 14336: 8 tokens 10.8 against 13.4, 32 15.9
// against 15.7, 48 21.0 against 17.0).
hipError_t launch_gated(const GatedForward& p, hipStream_t s) {
  Epilogue e{};
  e.nseg = 2;
  e.seg_end[0] = (int)p.f;
  e.a_scale = p.a_scale;
  e.ws_dev = p.scales;
  e.out = p.h;
  e.out_dtype = p.h_dtype;
  e.ldo = p.f;
  e.mid_dtype = WFB_F32;
  e.gate_up = p.gate_up;
  e.ldgu = 2 * gated_pad(p.f);
  const int n = (int)(2 * p.f), k = (int)p.k, m = (int)p.m;
  if (m <= 32 && !p.gate_up && p.f % 32 == 0 && (int64_t)n * (k / 4) <= INT32_MAX && (m - 1) * p.lda + k <= INT32_MAX)
    return launch_gemm_i2s_glu(p.qw, n, k, p.codes, m, p.lda, p.act, e, s);
  return launch_gemm_i2s_pair(p.qw, n, k, p.codes, m, p.lda, p.act, e, s);
}

int64_t gated_grad_workspace(const GatedGrad& p) { return grad_layout(p).bytes; }

hipError_t launch_gated_grad(const GatedGrad& p, void* work, hipStream_t s) {
  const GradLayout l = grad_layout(p);
  char* ws = static_cast<char*>(work);
  const int64_t esz = p.gh_dtype == WFB_F32 ? 16 : 8;
  const GradSrc src{p.gate_up, p.gh, p.ldg, (uintptr_t)p.gh % esz == 0 && p.ldg % 4 == 0, (int)p.m, (int)p.f, (int)l.fp,
                    p.scales, p.a_scale};
  auto* bx = reinterpret_cast<uint16_t*>(ws + l.bx);
  auto* bw = reinterpret_cast<uint16_t*>(ws + l.bw);
  Operands ops{};
  ops.qw = p.qw, ops.row_bytes = p.k_pad / 4;
  ops.codes = p.codes, ops.lda = p.lda, ops.vec = (uintptr_t)p.codes % 16 == 0 && p.lda % 16 == 0;
  ops.K = (int)p.k, ops.mp = (int)l.mp;
  ops.wt = l.px ? bx : nullptr, ops.ct = l.pw ? bw : nullptr;
  ops.top_rows = (int)l.top_rows, ops.top_tiles = (int)l.row_tiles, ops.tops = (int)(l.row_tiles * l.col_tiles);
  ops.weight_tiles = (int)(2 * l.fp / 64), ops.weights = l.px ? ops.weight_tiles * (int)((p.k + 127) / 128) : 0;
  ops.code_tiles = (int)(l.mp / 64);
  hipError_t e;
#define WFB_LAYOUTS(ACT)                                                               \
  (p.gh_dtype == WFB_F32    ? launch_layouts<ACT, WFB_F32>(src, ops, l, ws, s)        \
   : p.gh_dtype == WFB_BF16 ? launch_layouts<ACT, WFB_BF16>(src, ops, l, ws, s)       \
                            : launch_layouts<ACT, WFB_F16>(src, ops, l, ws, s))
  e = p.act == WFB_ACT_SILU ? WFB_LAYOUTS(WFB_ACT_SILU) : WFB_LAYOUTS(WFB_ACT_RELU2);
#undef WFB_LAYOUTS
  if (e != hipSuccess) return e;
  const float* inverse = reinterpret_cast<const float*>(ws + l.inverse);
  if (l.px) {
    GradGemm g{};
    g.a = reinterpret_cast<const uint16_t*>(ws + l.ax);
    g.lda = g.ldb = 2 * l.fp;
    g.a_plane = p.m * 2 * l.fp;
    g.b = bx;
    g.I = (int)p.m;
    g.J = (int)p.k;
    g.c_a = (int)(2 * l.fp);
    g.row_scale = inverse;
    g.out = p.gx;
    g.out_dtype = p.gx_dtype;
    g.ldo = p.k;
    if ((e = run_gemm16(g, l.plan_x, 2 * l.fp, reinterpret_cast<float*>(ws + l.parts_x), s)) != hipSuccess) return e;
  }
  if (l.pw) {
    GradGemm g{};
    g.a = reinterpret_cast<const uint16_t*>(ws + l.aw);
    g.lda = g.ldb = l.mp;
    g.a_plane = 2 * p.f * l.mp;
    g.b = bw;
    g.I = (int)(2 * p.f);
    g.J = (int)p.k;
    g.c_a = (int)l.mp;
    g.row_scale = inverse + p.m;
    g.out = p.gw;
    g.out_dtype = p.gw_dtype;
    g.ldo = p.k;
    if ((e = run_gemm16(g, l.plan_w, p.m, reinterpret_cast<float*>(ws + l.parts_w), s)) != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace wfb
