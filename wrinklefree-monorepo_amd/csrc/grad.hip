// Gradients of the ternary linear under the straight-through estimator, on the bf16 matrix cores.
//
// The reference trains F.linear(x + (q(x) - x).detach(), w + (q(w) - w).detach())
// (packages/training/src/wrinklefree/models/bitlinear.py:86-113), whose gradients are plain products with one
// exactly representable operand:
//   grad_x[m, k] = w_scale * sum_n g[m, n] * t[n, k]               t in {-1, 0, 1}
//   grad_w[n, k] = sum_m (g[m, n] * a_scale[m]) * q[m, k]          q an int8 code
// Both run as C[i, j] = alpha * sum_p sum_c A_p[i, c] * B[j, c] with bf16 operands and fp32 accumulators.  t and
// q are exact in bf16.  An fp32 factor enters as three bf16 planes cut off its bits (8 + 8 + 8 significant bits:
// the planes sum to the value exactly, see split3 for where), so every product is exact in fp32 and the only roundings
// are those of the fp32 sums and of g * a_scale (an fp32 product would round q * a_scale instead: where g * a_scale
// leaves fp32's range, a code of 0 gives NaN).  A bf16 gradient is its own single plane in grad_x.
//
// Bound by the matrix cores: one pass over grad_x and three over grad_w instead of fp32 products, which run at a
// sixteenth of the bf16 rate.  2048 tokens, 2560 -> 6912, bf16 (traced): grad_x 549 -> 87 us + 12 for its three
// partial sums, grad_w 549 -> 180 + 7 us, the layout kernels 40 us in place of 160 us of conversions and transposes;
// the whole step 1364 -> 397 us.
//
// Two steps.  Layout kernels write the operands with the summed index contiguous (the ternary codes and the int8
// codes transposed to bf16; g * a_scale transposed and split), zero-padded to whole stages; then the tile kernel.

#include <algorithm>

#include "grad_tile.h"

namespace wfb {

namespace {

// v = p[0] + p[1] + p[2] exactly for |v| above 2^-110 (below, bits under 2^-133, the smallest bf16, are cut off): each
// plane is the top 16 bits of what is left, by truncation, so none overflows and each remainder is exact.  An
// infinite v has the planes v, 0, 0 and a NaN NaN, 0, 0: they reach the product as they are.
__device__ __forceinline__ void split3(float v, uint16_t (&p)[3]) {
  const uint32_t u = __float_as_uint(v);
  const bool finite = (u & 0x7f800000u) != 0x7f800000u;
  const float h = __uint_as_float(u & 0xffff0000u);
  const float r1 = finite ? __fsub_rn(v, h) : 0.0f;
  const uint32_t u1 = __float_as_uint(r1);
  const float r2 = __fsub_rn(r1, __uint_as_float(u1 & 0xffff0000u));
  p[0] = (uint16_t)(u >> 16) | (uint16_t)(!finite && (u & 0x007fffffu) ? 0x40u : 0u);
  p[1] = (uint16_t)(u1 >> 16);
  p[2] = (uint16_t)(__float_as_uint(r2) >> 16);
}

// ---- operand layouts ---------------------------------------------------------------------------

// Planes of v[n][m] = g[m][n] * a_scale[m], dst[p][n][m] with rows of mp elements (m >= M: zeros).  One 64 x 64
// tile per workgroup through LDS: whole 128-byte lines in and out; the padded rows keep both sides of the
// transpose free of bank conflicts.  With colsum, also the tile's column sums of g, colsum[m0 / 64][n].
template <int DT>
__global__ __launch_bounds__(256) void grad_scaled_t_kernel(const void* __restrict__ g, int64_t ldg,
                                                            const float* __restrict__ a_scale, int64_t M, int64_t N,
                                                            int64_t mp, uint16_t* __restrict__ dst,
                                                            float* __restrict__ colsum) {
  __shared__ float tile[64][65];
  __shared__ float sums[4][64];
  const int64_t m0 = (int64_t)blockIdx.x * 64, n0 = (int64_t)blockIdx.y * 64;
  const int c = threadIdx.x & 63, r0 = threadIdx.x >> 6;
  float v[16], sum = 0.0f;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const int64_t m = m0 + r0 + 4 * j, n = n0 + c;
    const int64_t mc = m < M ? m : M - 1, nc = n < N ? n : N - 1;
    const float x = load_elem<DT>(g, mc * ldg + nc), s = a_scale[mc];
    v[j] = m < M ? __fmul_rn(x, s) : 0.0f;
    sum += m < M ? x : 0.0f;
  }
  sums[r0][c] = sum;
#pragma unroll
  for (int j = 0; j < 16; ++j) tile[r0 + 4 * j][c] = v[j];
  __syncthreads();
  if (colsum && r0 == 0 && n0 + c < N)
    colsum[(int64_t)blockIdx.x * N + n0 + c] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
  const int64_t plane = N * mp;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int idx = threadIdx.x + 256 * j, ch = idx & 7, nl = idx >> 3;
    const int64_t n = n0 + nl, m = m0 + 8 * ch;
    if (n >= N || m >= mp) continue;
    union { uint16_t h[8]; uint4 q; } o[3];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint16_t p[3];
      split3(tile[8 * ch + e][nl], p);
#pragma unroll
      for (int k = 0; k < 3; ++k) o[k].h[e] = p[k];
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(dst + k * plane + n * mp + m) = o[k].q;
  }
}

// Planes of g itself, dst[p][m][n] with rows of np elements (n >= N: zeros): three planes of an fp32 or fp16
// gradient, or one (a copy with padded rows) of a bf16 gradient whose rows do not start 16-byte aligned.
template <int DT, int P>
__global__ __launch_bounds__(256) void grad_planes_kernel(const void* __restrict__ g, int64_t ldg, int64_t M,
                                                          int64_t N, int64_t np, uint16_t* __restrict__ dst) {
  const int64_t per = np / 8, idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= M * per) return;
  const int64_t m = idx / per, n = 8 * (idx % per);
  union { uint16_t h[8]; uint4 q; } o[P];
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int64_t nc = n + e < N ? n + e : N - 1;
    v[e] = load_elem<DT>(g, m * ldg + nc);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    uint16_t p[3];
    split3(n + e < N ? v[e] : 0.0f, p);
#pragma unroll
    for (int k = 0; k < P; ++k) o[k].h[e] = p[k];
  }
#pragma unroll
  for (int k = 0; k < P; ++k) *reinterpret_cast<uint4*>(dst + k * M * np + m * np + n) = o[k].q;
}

// I2_S codes of W[n][k] as bf16 {-u, 0, u}, u = scale_unit(scale), dst[k][n], rows of np elements (n >= N: zeros).
// One 128-weight block of 64 rows per workgroup.
__global__ __launch_bounds__(256) void weight_codes_t_kernel(const uint8_t* __restrict__ qw, int64_t row_bytes,
                                                             int64_t N, int64_t K, int64_t np,
                                                             const float* __restrict__ scale,
                                                             uint16_t* __restrict__ dst) {
  __shared__ __attribute__((aligned(4))) uint8_t tile[64][36];
  const int64_t n0 = (int64_t)blockIdx.x * 64, b = blockIdx.y;
  {
    const int r = threadIdx.x >> 2, c8 = threadIdx.x & 3;  // 8 bytes of one row per thread
    const int64_t n = n0 + r;
    const uint2 w = *reinterpret_cast<const uint2*>(qw + (n < N ? n : N - 1) * row_bytes + 32 * b + 8 * c8);
    uint32_t* t = reinterpret_cast<uint32_t*>(&tile[r][8 * c8]);  // (code 1 = weight 0)
    t[0] = n < N ? w.x : 0x55555555u;
    t[1] = n < N ? w.y : 0x55555555u;
  }
  const float unit = scale_unit(scale[0]);
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int idx = threadIdx.x + 256 * it, ch = idx & 7, kl = idx >> 3;  // 8 rows n of column kl
    const int64_t k = 128 * b + kl, n = n0 + 8 * ch;
    if (k >= K || n >= np) continue;
    const int j = kl & 31, sh = 6 - 2 * (kl >> 5);
    union { uint16_t h[8]; uint4 q4; } o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int code = (tile[8 * ch + e][j] >> sh) & 3;
      o.h[e] = (uint16_t)(__float_as_uint((float)(code - 1) * unit) >> 16);
    }
    *reinterpret_cast<uint4*>(dst + k * np + n) = o.q4;
  }
}

// ---- tile kernel (grad_tile.h) -----------------------------------------------------------------

// Tile variants: workgroups a CU holds, the rate (PFLOP/s) with all of them busy and the microseconds a round of
// workgroups takes beside its products (first loads, epilogue), measured on MI355X.  Three planes run slower than
// one against ternary rows: the same kernel on constant data reaches 1.5 PFLOP/s, on random planes 1.15 -- the
// power that toggling operands draw lowers the clock.
constexpr Variant kVariants[] = {{1, 256, 256, 64, 1, 1.20, 8}, {1, 128, 128, 64, 2, 1.05, 5},
                                 {1, 64, 128, 64, 3, 0.80, 3}, {3, 128, 256, 32, 2, 1.15, 8},
                                 {3, 64, 128, 32, 4, 0.85, 2.5}};
constexpr int kNumVariants = sizeof(kVariants) / sizeof(kVariants[0]);

Plan plan(int planes, int64_t I, int64_t J, int64_t C) { return plan_of(kVariants, kNumVariants, planes, I, J, C); }

hipError_t run_gemm(GradGemm p, const Plan& pl, int64_t C, float* parts, hipStream_t s) {
  set_plan(p, pl, kVariants, C, parts);
  switch (pl.variant) {  // kVariants
    case 0: return launch_tiles<false, 1, 4, 2, 2, 4, 64, 2>(p, pl, s);
    case 1: return launch_tiles<false, 1, 2, 2, 2, 2, 64, 2>(p, pl, s);
    case 2: return launch_tiles<false, 1, 1, 2, 2, 2, 64, 3>(p, pl, s);
    case 3: return launch_tiles<false, 3, 2, 4, 2, 2, 32, 2>(p, pl, s);
    default: return launch_tiles<false, 3, 1, 2, 2, 2, 32, 4>(p, pl, s);
  }
}

int64_t part_bytes(const Plan& pl) { return part_bytes_of(kVariants, pl); }

int grad_x_planes(int gdt) { return gdt == WFB_BF16 ? 1 : 3; }

}  // namespace

// grad_x operands in the workspace: [K][Np] weight codes, then the planes of g (always reserved, so that the size
// does not depend on the alignment of g), then the partial sums.
int64_t grad_x_workspace(int64_t m, int64_t n, int64_t k, int gdt) {
  const int64_t np = pad_to(n, kPad);
  const int P = grad_x_planes(gdt);
  return align256(2 * k * np) + align256(2 * P * m * np) + part_bytes(plan(P, m, k, n));
}

int64_t grad_w_workspace(int64_t m, int64_t n, int64_t k) {
  const int64_t mp = pad_to(m, kPad);
  return align256(2 * 3 * n * mp) + align256(2 * k * mp) + align256(4 * (mp / 64) * n) +
         part_bytes(plan(3, n, k, m));
}

void grad_plan(bool of_x, int64_t m, int64_t n, int64_t k, int gdt, int64_t (&out)[5]) {
  const Plan pl = of_x ? plan(grad_x_planes(gdt), m, k, n) : plan(3, n, k, m);
  const Variant& v = kVariants[pl.variant];
  const int64_t o[5] = {v.bi, v.bj, pl.tiles, pl.full, pl.nsplit};
  std::copy(o, o + 5, out);
}

hipError_t launch_grad_x(const void* g, int gdt, int64_t ldg, int64_t m, int64_t n, const uint8_t* qw, int64_t k,
                         int64_t k_pad, const float* w_scale, void* out, int odt, int64_t ldo, void* work,
                         hipStream_t s) {
  const int64_t np = pad_to(n, kPad);
  const int P = grad_x_planes(gdt);
  char* ws = static_cast<char*>(work);
  uint16_t* wt = reinterpret_cast<uint16_t*>(ws);
  uint16_t* gp = reinterpret_cast<uint16_t*>(ws + align256(2 * k * np));
  float* parts = reinterpret_cast<float*>(ws + align256(2 * k * np) + align256(2 * P * m * np));
  hipLaunchKernelGGL(weight_codes_t_kernel, dim3((unsigned)(np / 64), (unsigned)((k + 127) / 128)), dim3(256), 0, s, qw,
                     k_pad / 4, n, k, np, w_scale, wt);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  GradGemm p{};
  p.b = wt;
  p.ldb = np;
  p.I = (int)m;
  p.J = (int)k;
  p.alpha = w_scale;
  p.out = out;
  p.out_dtype = odt;
  p.ldo = ldo;
  if (gdt == WFB_BF16 && (uintptr_t)g % 16 == 0 && ldg % 8 == 0 && n % 8 == 0) {
    p.a = static_cast<const uint16_t*>(g);
    p.lda = ldg;
    p.c_a = (int)n;
  } else {
    const unsigned grid = (unsigned)((m * (np / 8) + 255) / 256);
    if (gdt == WFB_BF16)
      hipLaunchKernelGGL((grad_planes_kernel<WFB_BF16, 1>), dim3(grid), dim3(256), 0, s, g, ldg, m, n, np, gp);
    else if (gdt == WFB_F32)
      hipLaunchKernelGGL((grad_planes_kernel<WFB_F32, 3>), dim3(grid), dim3(256), 0, s, g, ldg, m, n, np, gp);
    else
      hipLaunchKernelGGL((grad_planes_kernel<WFB_F16, 3>), dim3(grid), dim3(256), 0, s, g, ldg, m, n, np, gp);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    p.a = gp;
    p.lda = np;
    p.a_plane = m * np;
    p.c_a = (int)np;
  }
  return run_gemm(p, plan(P, m, k, n), n, parts, s);
}

hipError_t launch_grad_w(const void* g, int gdt, int64_t ldg, int64_t m, int64_t n, const int8_t* q, int64_t ldq,
                         const float* a_scale, int64_t k, void* out, int odt, int64_t ldo, void* bias_out, int bdt,
                         void* work, hipStream_t s) {
  const int64_t mp = pad_to(m, kPad);
  char* ws = static_cast<char*>(work);
  uint16_t* gt = reinterpret_cast<uint16_t*>(ws);
  uint16_t* qt = reinterpret_cast<uint16_t*>(ws + align256(2 * 3 * n * mp));
  float* sums = reinterpret_cast<float*>(ws + align256(2 * 3 * n * mp) + align256(2 * k * mp));
  float* parts = reinterpret_cast<float*>(reinterpret_cast<char*>(sums) + align256(4 * (mp / 64) * n));
  float* cs = bias_out ? sums : nullptr;
  const dim3 gg((unsigned)(mp / 64), (unsigned)((n + 63) / 64));
  if (gdt == WFB_F32)
    hipLaunchKernelGGL((grad_scaled_t_kernel<WFB_F32>), gg, dim3(256), 0, s, g, ldg, a_scale, m, n, mp, gt, cs);
  else if (gdt == WFB_BF16)
    hipLaunchKernelGGL((grad_scaled_t_kernel<WFB_BF16>), gg, dim3(256), 0, s, g, ldg, a_scale, m, n, mp, gt, cs);
  else
    hipLaunchKernelGGL((grad_scaled_t_kernel<WFB_F16>), gg, dim3(256), 0, s, g, ldg, a_scale, m, n, mp, gt, cs);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (bias_out && (e = launch_column_sum(sums, (int)(mp / 64), n, bias_out, bdt, s)) != hipSuccess) return e;
  const dim3 gq((unsigned)(mp / 64), (unsigned)((k + 63) / 64));
  if ((uintptr_t)q % 16 == 0 && ldq % 16 == 0)
    hipLaunchKernelGGL((codes_t_kernel<true>), gq, dim3(256), 0, s, q, ldq, m, k, mp, qt);
  else
    hipLaunchKernelGGL((codes_t_kernel<false>), gq, dim3(256), 0, s, q, ldq, m, k, mp, qt);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  GradGemm p{};
  p.a = gt;
  p.lda = mp;
  p.a_plane = n * mp;
  p.b = qt;
  p.ldb = mp;
  p.I = (int)n;
  p.J = (int)k;
  p.c_a = (int)mp;
  p.out = out;
  p.out_dtype = odt;
  p.ldo = ldo;
  return run_gemm(p, plan(3, n, k, m), m, parts, s);
}

}  // namespace wfb
