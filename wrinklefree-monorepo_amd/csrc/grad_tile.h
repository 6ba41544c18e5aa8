// The matrix-core product of the gradient passes: C[i, j] = alpha * sum_p sum_c A_p[i, c] B[j, c] of bf16 or fp16 operands with
// fp32 sums, and the plan of its tiles (grad.hip, gated.hip).
#pragma once

#include "wfb_common.h"

namespace wfb {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

typedef float f32x4_t __attribute__((ext_vector_type(4)));

template <bool F16>
struct Op16 {
  typedef bf16x8_t v8;
  static __device__ __forceinline__ f32x16_t mfma(v8 a, v8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Op16<true> {
  typedef f16x8_t v8;
  static __device__ __forceinline__ f32x16_t mfma(v8 a, v8 b, f32x16_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t mfma16(v8 a, v8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// The weight scale's power of two, 2^-126 at least; 1 for a scale that is not finite.  The weight codes
// carry it (exact in bf16), so the sums of a gradient run at the size of its result, and the epilogue's factor is what
// is left of the scale: the same bits, without overflow where only the unscaled sum leaves fp32's range.
__device__ __forceinline__ float scale_unit(float s) {
  const uint32_t e = __float_as_uint(s) & 0x7f800000u;
  return e == 0x7f800000u ? 1.0f : __uint_as_float(e ? e : 0x00800000u);
}

// int8 codes q[m][k] as bf16 or fp16 (both exact) dst[k][m], rows of mp elements (m >= M: zeros).  VEC: 16 codes per load (rows 16-byte
// aligned); a row's last codes, fewer than 16, one at a time: nothing has to lie behind the last row's.
template <bool VEC, bool F16>
__device__ __forceinline__ void codes_t(const int8_t* __restrict__ q, int64_t ldq, int64_t M, int64_t K, int64_t mp, int bx,
                                        int by, uint16_t* __restrict__ dst, int8_t (&tile)[64][68]) {
  const int64_t m0 = (int64_t)bx * 64, k0 = (int64_t)by * 64;
  const int r = threadIdx.x >> 2, c = 16 * (threadIdx.x & 3);  // 16 codes of row r
  const int64_t m = m0 + r, row = (m < M ? m : M - 1) * ldq;
  uint32_t v[4] = {0, 0, 0, 0};
  if (VEC && k0 + c + 16 <= K) {
    if (m < M) {
      const uint4 x = *reinterpret_cast<const uint4*>(q + row + k0 + c);
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    }
  } else if (k0 + c < K) {
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t k = k0 + c + e;
      const uint32_t b = (uint8_t)q[row + (k < K ? k : K - 1)];
      v[e / 4] |= (m < M ? b : 0u) << (8 * (e % 4));
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(&tile[r][c + 4 * e]) = v[e];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int idx = threadIdx.x + 256 * j, ch = idx & 7, kl = idx >> 3;
    const int64_t k = k0 + kl, mo = m0 + 8 * ch;
    if (k >= K || mo >= mp) continue;
    union { uint16_t h[8]; uint4 q4; } o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = (float)tile[8 * ch + e][kl];
      o.h[e] = F16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : (uint16_t)(__float_as_uint(v) >> 16);
    }
    *reinterpret_cast<uint4*>(dst + k * mp + mo) = o.q4;
  }
}

template <bool VEC>
__global__ __launch_bounds__(256) void codes_t_kernel(const int8_t* __restrict__ q, int64_t ldq, int64_t M, int64_t K,
                                                      int64_t mp, uint16_t* __restrict__ dst) {
  __shared__ __attribute__((aligned(4))) int8_t tile[64][68];
  codes_t<VEC, false>(q, ldq, M, K, mp, blockIdx.x, blockIdx.y, dst, tile);
}

typedef __attribute__((address_space(3))) void lds_void;
__device__ __forceinline__ void lds_load16(buf_t r, void* lds_base, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)lds_base, 16, voff, 0, 0, 0);
}

struct GradGemm {
  const uint16_t* a;   // [P][I][lda]
  int64_t lda, a_plane;
  const uint16_t* b;   // [J][ldb]
  int64_t ldb;
  int I, J;
  int c_a;             // elements of an A row (offsets past it read zeros)
  int stages;          // of BK elements, all splits together
  int full;            // the first `full` tiles are summed by one workgroup each,
  int nsplit;          // the others by nsplit: split s takes stages [s * per, ...), per = ceil(stages / nsplit)
  const float* alpha;  // device scalar, of which the B rows carry scale_unit, or null (1)
  const float* row_scale;  // (fp16 operands) [I], what row i of the product is multiplied by
  float* parts;        // fp32 partial tiles [tiles past full][nsplit][BI][BJ]
  void* out;           // [I][ldo] in out_dtype
  int out_dtype;
  int64_t ldo;
  bool vec;            // rows of out 16-byte aligned
};

__device__ __forceinline__ float alpha_of(const GradGemm& p) {
  if (!p.alpha) return 1.0f;
  const float s = p.alpha[0];
  return __fdiv_rn(s, scale_unit(s));  // (exact)
}

__device__ __forceinline__ void store1(const GradGemm& p, int64_t off, float y) {
  if (p.out_dtype == WFB_F32) reinterpret_cast<float*>(p.out)[off] = y;
  else if (p.out_dtype == WFB_BF16) reinterpret_cast<uint16_t*>(p.out)[off] = f32_to_bf16_rne(y);
  else reinterpret_cast<uint16_t*>(p.out)[off] = __builtin_bit_cast(uint16_t, (_Float16)y);
}

// 8 consecutive outputs at element offset off, column col
__device__ __forceinline__ void store8(const GradGemm& p, int64_t off, int col, float4 ya, float4 yb) {
  const float y[8] = {ya.x, ya.y, ya.z, ya.w, yb.x, yb.y, yb.z, yb.w};
  if (!p.vec || col + 8 > p.J) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < p.J) store1(p, off + e, y[e]);
    return;
  }
  if (p.out_dtype == WFB_F32) {
    float* o = reinterpret_cast<float*>(p.out) + off;
    *reinterpret_cast<float4*>(o) = ya;
    *reinterpret_cast<float4*>(o + 4) = yb;
    return;
  }
  union { uint16_t h[8]; uint4 q; } o;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    o.h[e] = p.out_dtype == WFB_BF16 ? f32_to_bf16_rne(y[e]) : __builtin_bit_cast(uint16_t, (_Float16)y[e]);
  *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + off) = o.q;
}

// C tile of (32 TI WI) x (32 TJ WJ), WI x WJ waves of (32 TI) x (32 TJ), v_mfma_f32_32x32x16_bf16 with B rows as
// src0 and A rows as src1 (lane (i, g), register r: row i of A, row 8 (r / 4) + 4 g + r % 4 of B).  The summed
// index advances in stages of BK: the P planes' rows and the B rows of a stage go from global memory straight
// into one of two LDS buffers (whole 64- or 128-byte row pieces, 16-byte chunks XOR-swizzled by row so that 16
// rows at one chunk meet 16 distinct bank groups), the next stage's loads in flight while a stage is multiplied.
// ST = 3, 4: a ring of so many buffers instead, ST - 1 stages in flight (see below), and v_mfma_f32_16x16x32 (lane (i, g),
// register r: row i of A, row 4 g + r of B).  Its sums are read and written half as often for a product as the 32 x 32
// form's, and large products are bound by the card's power: with operands out of cache 4096 x 2560 x 13824 302 -> 276 us,
// 28672 x 4096 x 2048 456 -> 416, 13824 x 2560 x 4096 in two planes 464 -> 427 (1.36 PFLOP/s) with it.  A wave's 64 x 128
// or 128 x 64 is better than 128 x 128 with half the waves (416 against 493): two waves of a SIMD cover each other's waits.
template <bool F16, int P, int TI, int TJ, int WI, int WJ, int BK, int WPE, int ST = 2>
__global__ __launch_bounds__(64 * WI * WJ) __attribute__((amdgpu_waves_per_eu(WPE, WPE))) void grad_tile_kernel(
    GradGemm p, int tiles_i, int tiles_j) {
  constexpr int W = WI * WJ, BI = 32 * TI * WI, BJ = 32 * TJ * WJ;
  constexpr int ROW = 2 * BK, CH = ROW / 16, RPI = 64 / CH;  // bytes and chunks of a row, rows per load
  constexpr int ASZ = P * BI * ROW, BSZ = BJ * ROW, SZ = ASZ + BSZ;
  constexpr int AI = ASZ / 1024 / W, NB = BSZ / 1024 / W;
  constexpr int KS = BK / 16;
  static_assert(AI * 1024 * W == ASZ && NB * 1024 * W == BSZ && (BK == 32 || BK == 64), "tile shape");
  static_assert((P * BI / RPI / W) * W * RPI == P * BI && BI % RPI == 0, "a load stays in one plane");
  __shared__ __attribute__((aligned(16))) uint8_t lds0[SZ];
  __shared__ __attribute__((aligned(16))) uint8_t lds1[SZ];
  __shared__ __attribute__((aligned(16))) uint8_t lds2[ST > 2 ? SZ : 16];
  __shared__ __attribute__((aligned(16))) uint8_t lds3[ST > 3 ? SZ : 16];
  const int tid = threadIdx.x, l = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = w / WJ, wj = w % WJ, i = l & 31, g = l >> 5;

  // whole tiles first, each XCD a contiguous range of them; then the split ones
  const int per8 = (p.full + 7) / 8, bid = blockIdx.x, u = bid - 8 * per8;
  const bool whole = u < 0;
  const int tt = whole ? (bid % 8) * per8 + bid / 8 : p.full + u / p.nsplit;
  if (whole && tt >= p.full) return;
  const int split = whole ? 0 : u % p.nsplit;
  constexpr int kGroup = 8;
  const int gsz = kGroup * tiles_j, grp = tt / gsz, rr = tt - grp * gsz;
  const int gm = min(kGroup, tiles_i - grp * kGroup);
  const int i0 = __builtin_amdgcn_readfirstlane((grp * kGroup + rr % gm) * BI);
  const int j0 = __builtin_amdgcn_readfirstlane((rr / gm) * BJ);
  const int per = whole ? p.stages : (p.stages + p.nsplit - 1) / p.nsplit;
  const int s0 = __builtin_amdgcn_readfirstlane(split * per), s1 = __builtin_amdgcn_readfirstlane(min(s0 + per, p.stages));

  const int irows = min(BI, p.I - i0), jrows = min(BJ, p.J - j0);
  const uint32_t a_row = 2u * (uint32_t)p.lda, b_row = 2u * (uint32_t)p.ldb;
  const uint32_t a_end = (uint32_t)irows * a_row, b_end = (uint32_t)jrows * b_row;
  buf_t ab[AI];  // of the plane that load jj of this wave lies in
#pragma unroll
  for (int jj = 0; jj < AI; ++jj)
    ab[jj] = make_buf(p.a + (RPI * (AI * w + jj) / BI) * p.a_plane + (int64_t)i0 * p.lda, a_end);
  const buf_t bb = make_buf(p.b + (int64_t)j0 * p.ldb, b_end);
  const uint32_t a_cols = 2u * (uint32_t)p.c_a;

  auto swz = [](int r) { return BK == 64 ? ((r >> 1) & 7) : ((r >> 2) & 3); };
  // rows past the operand lie past the buffer's end and read zeros
  uint32_t arow[AI], acol[AI], boff[NB];
#pragma unroll
  for (int jj = 0; jj < AI; ++jj) {
    const int R = RPI * (AI * w + jj) + l / CH, r = R % BI;
    arow[jj] = (uint32_t)r * a_row;
    acol[jj] = 16u * ((l % CH) ^ swz(r));
  }
#pragma unroll
  for (int jj = 0; jj < NB; ++jj) {
    const int r = RPI * (NB * w + jj) + l / CH;
    boff[jj] = (uint32_t)r * b_row + 16u * ((l % CH) ^ swz(r));
  }
  auto issue = [&](int s, uint8_t* lds) {
#pragma unroll
    for (int jj = 0; jj < AI; ++jj) {
      const uint32_t col = (uint32_t)ROW * s + acol[jj];
      lds_load16(ab[jj], lds + (AI * w + jj) * 1024, col < a_cols ? arow[jj] + col : a_end);
    }
#pragma unroll
    for (int jj = 0; jj < NB; ++jj) lds_load16(bb, lds + ASZ + (NB * w + jj) * 1024, boff[jj] + (uint32_t)ROW * s);
  };

  constexpr bool kRing = ST > 2;
  f32x16_t acc[kRing ? 1 : TJ][kRing ? 1 : TI];
  f32x4_t acc4[kRing ? 2 * TJ : 1][kRing ? 2 * TI : 1];
  if constexpr (kRing) {
#pragma unroll
    for (int tj = 0; tj < 2 * TJ; ++tj)
#pragma unroll
      for (int ti = 0; ti < 2 * TI; ++ti) acc4[tj][ti] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  } else {
#pragma unroll
    for (int tj = 0; tj < TJ; ++tj)
#pragma unroll
      for (int ti = 0; ti < TI; ++ti)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[tj][ti][q] = 0.0f;
  }

  typedef typename Op16<F16>::v8 v8;
  if constexpr (kRing) {
    // Stage s: the loads of stage s + ST - 1 go into the buffer of stage s - 1, which every wave had read before the
    // barrier at that stage's end.  Its own end waits, in every wave, until its reads of cur are done and all but the
    // last ST - 2 stages' loads of this wave have landed, then for the others.  The count is fixed: stages past s1 are
    // issued too, from past the operands' ends (zeros, no traffic).
    constexpr int kOpen = (ST - 2) * (AI + NB), kWait = (kOpen & 15) | 0x70 | (kOpen >> 4 << 14);  // vmcnt, lgkmcnt(0)
    static_assert(kOpen < 64, "vmcnt's range");
    // loads [from, to) of a stage's AI + NB
    auto load = [&](int s, uint8_t* lds, int from, int to) {
      const bool on = s < s1;
#pragma unroll
      for (int jj = 0; jj < AI; ++jj) {
        if (jj < from || jj >= to) continue;
        const uint32_t col = (uint32_t)ROW * s + acol[jj];
        lds_load16(ab[jj], lds + (AI * w + jj) * 1024, on && col < a_cols ? arow[jj] + col : a_end);
      }
#pragma unroll
      for (int jj = 0; jj < NB; ++jj) {
        if (AI + jj < from || AI + jj >= to) continue;
        lds_load16(bb, lds + ASZ + (NB * w + jj) * 1024, on ? boff[jj] + (uint32_t)ROW * s : b_end);
      }
    };
    auto meet = [&] {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (orders the LDS accesses for the compiler)
      __builtin_amdgcn_s_waitcnt(kWait);
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    // A step is 64 rows of a plane of A by 32 elements: 4 fragments, read during the step before.  B's fragments of 32
    // elements serve all steps over them, and each is overwritten behind its last use.
    constexpr int NA = P * TI / 2, KS = BK / 32 * NA, M = 8 * TJ;
    static_assert(TI % 2 == 0 && KS % 2 == 0, "a stage starts with fragment set 0");
    constexpr int LP = (AI + NB + KS - 1) / KS;  // loads that go with one step's products
    const int i4 = l & 15, g4 = l >> 4;
    const uint32_t afr = (uint32_t)(wi * TI * 32 + i4) * ROW, bfr = ASZ + (uint32_t)(wj * TJ * 32 + i4) * ROW;
    v8 af[2][4], bf[2 * TJ];
    auto chunk = [&](int k) { return (uint32_t)(((4 * k + g4) ^ swz(i4)) * 16); };
    auto read_a = [&](const uint8_t* lds, int x) {
      const int n = x % NA, q = n / (TI / 2), t = n % (TI / 2);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        af[x & 1][e] = *reinterpret_cast<const v8*>(lds + afr + (q * BI + 64 * t + 16 * e) * ROW + chunk(x / NA));
    };
    auto read_b = [&](const uint8_t* lds, int k, int tj) {
      bf[tj] = *reinterpret_cast<const v8*>(lds + bfr + 16 * tj * ROW + chunk(k));
    };
    // step x of a stage, the reads for the next one from lds and `loads` loads among its products
    auto step = [&](int x, bool reads, const uint8_t* lds, int loads) __attribute__((always_inline)) {
      const int nx = (x + 1) % KS, t = x % (TI / 2);
      const bool turn = (x + 1) % NA == 0;
      if (reads) read_a(lds, nx);
#pragma unroll
      for (int tj = 0; tj < 2 * TJ; ++tj) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc4[tj][4 * t + e] = Op16<F16>::mfma16(bf[tj], af[x & 1][e], acc4[tj][4 * t + e]);
        if (reads && turn) read_b(lds, nx / NA, tj);
      }
#pragma unroll
      for (int k = 0; k < M; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (reads && k < 4) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        if (reads && turn && k % 4 == 3) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        if (loads && k * loads / M != (k + 1) * loads / M) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    // stage s from cur, behind the last step of stage s - 1
    auto ring = [&](int s, uint8_t* cur, uint8_t* last) __attribute__((always_inline)) {
      meet();
      load(s + ST - 1, last, 0, LP);
      step(KS - 1, true, cur, LP);
#pragma unroll
      for (int x = 0; x + 1 < KS; ++x) {
        load(s + ST - 1, last, LP * (x + 1), LP * (x + 2));
        step(x, true, cur, max(min(AI + NB - LP * (x + 1), LP), 0));
      }
    };
    uint8_t* const b2 = ST > 2 ? lds2 : lds0;
    uint8_t* const b3 = ST > 3 ? lds3 : lds0;
    if (s0 < s1) {
      load(s0, lds0, 0, AI + NB);
      load(s0 + 1, lds1, 0, AI + NB);
      if constexpr (ST > 3) load(s0 + 2, b2, 0, AI + NB);
      meet();
      read_a(lds0, 0);
#pragma unroll
      for (int tj = 0; tj < 2 * TJ; ++tj) read_b(lds0, 0, tj);
      load(s0 + ST - 1, ST > 3 ? b3 : b2, 0, AI + NB);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x + 1 < KS; ++x) step(x, true, lds0, 0);
      // (whole turns of the ring, then what is left: a loop that could end within a turn would have the compiler lose
      // count of the loads in flight and wait for all of them once a turn)
      int s = s0 + 1;
      if constexpr (ST == 3) {
        for (; s + 3 <= s1; s += 3) {
          ring(s, lds1, lds0);
          ring(s + 1, b2, lds1);
          ring(s + 2, lds0, b2);
        }
        if (s < s1) ring(s, lds1, lds0);
        if (s + 1 < s1) ring(s + 1, b2, lds1);
      } else {
        for (; s + 4 <= s1; s += 4) {
          ring(s, lds1, lds0);
          ring(s + 1, b2, lds1);
          ring(s + 2, b3, b2);
          ring(s + 3, lds0, b3);
        }
        if (s < s1) ring(s, lds1, lds0);
        if (s + 1 < s1) ring(s + 1, b2, lds1);
        if (s + 2 < s1) ring(s + 2, b3, b2);
      }
      step(KS - 1, false, lds0, 0);
      __builtin_amdgcn_s_waitcnt(0x0F70);  // the last stages' zeros: the buffers are the epilogue's from here on
    }
  } else {
    const uint32_t afr = (uint32_t)(wi * TI * 32 + i) * ROW, bfr = ASZ + (uint32_t)(wj * TJ * 32 + i) * ROW;
    // fragments of one 16-element step, two sets: a step's MFMAs run while the next step's are read
    v8 af[2][P][TI], bf[2][TJ];
    auto read = [&](const uint8_t* lds, int x) {
      const uint32_t c = (uint32_t)(((2 * x + g) ^ swz(i)) * 16);
#pragma unroll
      for (int tj = 0; tj < TJ; ++tj) bf[x & 1][tj] = *reinterpret_cast<const v8*>(lds + bfr + tj * 32 * ROW + c);
#pragma unroll
      for (int q = 0; q < P; ++q)
#pragma unroll
        for (int ti = 0; ti < TI; ++ti)
          af[x & 1][q][ti] = *reinterpret_cast<const v8*>(lds + afr + (q * BI + ti * 32) * ROW + c);
    };
    auto multiply = [&](int x, bool reads, int loads = 0) {
#pragma unroll
      for (int q = 0; q < P; ++q)
#pragma unroll
        for (int ti = 0; ti < TI; ++ti)
#pragma unroll
          for (int tj = 0; tj < TJ; ++tj)
            acc[tj][ti] = Op16<F16>::mfma(bf[x & 1][tj], af[x & 1][q][ti], acc[tj][ti]);
      // the reads spread over the MFMAs (left alone, the compiler reads each fragment right before its first use
      // and waits for it)
#pragma unroll
      for (int k = 0; k < P * TI * TJ; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (reads && k < TJ + P * TI) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        if (loads && k * loads / (P * TI * TJ) != (k + 1) * loads / (P * TI * TJ))
          __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    // stage s from cur; its last step's MFMAs run behind the barrier that hands cur over to stage s + 2's loads and
    // behind the first reads of stage s + 1 from nxt
    auto stage = [&](int s, uint8_t* cur, uint8_t* nxt) {
#pragma unroll
      for (int x = 0; x + 1 < KS; ++x) {
        read(cur, x + 1);
        multiply(x, true);
      }
      if (s + 1 < s1) {
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's loads of stage s + 1 are in LDS
        __syncthreads();                      // everyone's, and everyone has read the last of stage s
        if (s + 2 < s1) issue(s + 2, cur);
        read(nxt, 0);
      }
      multiply(KS - 1, true);
    };
    static_assert(KS % 2 == 0, "a stage starts with fragment set 0");
    if (s0 < s1) {
      issue(s0, lds0);
      __builtin_amdgcn_s_waitcnt(0x0F70);
      __syncthreads();
      if (s0 + 1 < s1) issue(s0 + 1, lds1);
      read(lds0, 0);
      __builtin_amdgcn_sched_barrier(0);
      for (int s = s0; s < s1; s += 2) {
        stage(s, lds0, lds1);
        if (s + 1 < s1) stage(s + 1, lds1, lds0);
      }
    }
  }
  __syncthreads();  // the operand buffers are free

  // per 32-row MFMA tile: 32 rows x 32 TS fp32 (TS of the TJ tiles at a time, as the operand buffers hold it for
  // every wave) through this wave's LDS, 16-byte chunks XOR-swizzled by row; then 8 consecutive outputs of a row
  // per lane, whole lines per instruction
  constexpr int TS = 2 * (SZ / (4096 * TJ)) >= W ? TJ : TJ / 2;
  constexpr int CPR = 8 * TS, STG = 32 * CPR * 16;  // chunks of a staged row, bytes a wave stages
  constexpr int WPB = SZ / STG;                     // waves whose staging fits one buffer
  static_assert(TJ % TS == 0 && WPB >= 1 && 2 * WPB >= W, "staging fits the two operand buffers");
  uint8_t* st = w < WPB ? lds0 + w * STG : lds1 + (w - WPB) * STG;
  float alpha = whole ? alpha_of(p) : 1.0f;
  constexpr int LPR = CPR / 2, RP = 64 / LPR;
  float* const part = whole ? nullptr : p.parts + (int64_t)u * (BI * BJ);
  auto wave_sync = [] {  // orders the wave's LDS accesses for the compiler (the LDS keeps a wave's order by itself)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
#pragma unroll
  for (int ti = 0; ti < TI; ++ti) {
    auto scale_of = [&](int r) { return whole ? p.row_scale[min(i0 + wi * 32 * TI + ti * 32 + r, p.I - 1)] : 1.0f; };
    float alpha4[2];
    if constexpr (kRing) alpha4[0] = scale_of(l & 15), alpha4[1] = scale_of(16 + (l & 15));
    else if constexpr (F16) alpha = scale_of(i);
#pragma unroll
    for (int ts = 0; ts < TJ; ts += TS) {
      if constexpr (kRing) {
#pragma unroll
        for (int tj = 0; tj < 2 * TS; ++tj)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const f32x4_t& v = acc4[2 * ts + tj][2 * ti + h];
            const int r = 16 * h + (l & 15), c = 4 * tj + (l >> 4);
            *reinterpret_cast<float4*>(st + (r * CPR + (c ^ (r & (CPR - 1)))) * 16) =
                make_float4(v[0] * alpha4[h], v[1] * alpha4[h], v[2] * alpha4[h], v[3] * alpha4[h]);
          }
      } else {
#pragma unroll
        for (int tj = 0; tj < TS; ++tj)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const f32x16_t& v = acc[ts + tj][ti];
            const int c = tj * 8 + 2 * q + g;
            *reinterpret_cast<float4*>(st + (i * CPR + (c ^ (i & (CPR - 1)))) * 16) =
                make_float4(v[4 * q] * alpha, v[4 * q + 1] * alpha, v[4 * q + 2] * alpha, v[4 * q + 3] * alpha);
          }
      }
      wave_sync();
      constexpr int kStores = F16 ? 2 : 32 / RP;  // unrolled: whole, the stores' code is several times the products'
#pragma unroll kStores
      for (int jj = 0; jj < 32 / RP; ++jj) {
        const int r = RP * jj + l / LPR, c8 = l % LPR;
        const float4 ya = *reinterpret_cast<const float4*>(st + (r * CPR + ((2 * c8) ^ (r & (CPR - 1)))) * 16);
        const float4 yb = *reinterpret_cast<const float4*>(st + (r * CPR + ((2 * c8 + 1) ^ (r & (CPR - 1)))) * 16);
        const int row = wi * 32 * TI + ti * 32 + r, col = (wj * TJ + ts) * 32 + 8 * c8;  // within the tile
        if (!whole) {
          float4* o = reinterpret_cast<float4*>(part + row * BJ + col);
          o[0] = ya;
          o[1] = yb;
        } else if (i0 + row < p.I && j0 + col < p.J) {
          store8(p, (int64_t)(i0 + row) * p.ldo + j0 + col, j0 + col, ya, yb);
        }
      }
      wave_sync();
    }
  }
}

// The tiles past p.full: out = alpha * the sum of a tile's parts, in order.  A workgroup sums 2048 outputs.
template <bool F16>
__global__ __launch_bounds__(256) void grad_reduce_kernel(GradGemm p, int bi, int bj, int tiles_i, int tiles_j) {
  const int per = bi * bj / 2048, tile = blockIdx.x / per, e = 2048 * (blockIdx.x % per) + 8 * threadIdx.x;
  const int tt = p.full + tile, gsz = 8 * tiles_j, grp = tt / gsz, rr = tt - grp * gsz;  // the tile kernel's order
  const int gm = min(8, tiles_i - grp * 8);
  const int row = (grp * 8 + rr % gm) * bi + e / bj, col = (rr / gm) * bj + e % bj;
  if (row >= p.I || col >= p.J) return;
  const float* src = p.parts + (int64_t)tile * p.nsplit * (bi * bj) + e;
  float4 a = *reinterpret_cast<const float4*>(src), b = *reinterpret_cast<const float4*>(src + 4);
  for (int s = 1; s < p.nsplit; ++s) {
    src += bi * bj;
    const float4 c = *reinterpret_cast<const float4*>(src), d = *reinterpret_cast<const float4*>(src + 4);
    a.x += c.x, a.y += c.y, a.z += c.z, a.w += c.w;
    b.x += d.x, b.y += d.y, b.z += d.z, b.w += d.w;
  }
  const float alpha = F16 ? p.row_scale[row] : alpha_of(p);
  store8(p, (int64_t)row * p.ldo + col, col, make_float4(a.x * alpha, a.y * alpha, a.z * alpha, a.w * alpha),
         make_float4(b.x * alpha, b.y * alpha, b.z * alpha, b.w * alpha));
}

constexpr int64_t kPad = 64;  // operand rows are whole stages of every variant
constexpr int64_t pad_to(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

// A tile form: workgroups a CU holds, the rate (PFLOP/s) with all of them busy and the microseconds a round of workgroups
// takes beside its products (first loads, epilogue).
struct Variant {
  int planes, bi, bj, bk, per_cu;
  double rate, round_us;
  double partial = 0.85;  // (one workgroup a CU) a round that leaves CUs idle, of a full one's time
};

// The first `full` tiles whole, the others in nsplit parts of the summed index, each a workgroup of its own.
struct Plan {
  int variant;
  int64_t tiles, full;
  int nsplit;
};

// The least estimated time of every variant, of its tiles all split (or none) or only those past the last full round
// of workgroups, and of the number of parts: rounds of workgroups (a last round that leaves CUs with one workgroup
// runs it in less than the time of a full one) and the partial sums written and read back.  Swept on MI355X over
// every (variant, split of all tiles) of 18 shapes from 1 x 576 x 576 to 4096^3, both products: the estimate's pick
// is within 8% of the fastest on all but four, within 15% there.  Splitting only the tiles past the last full round
// (28 of 540 at 2048 x 6912 x 2560) took grad_w there from 200 us and 26 for all tiles' sums to 180-189 and 7.
// split_us: what each further part costs beside its traffic, the summing kernel's chain of loads.
inline Plan plan_of(const Variant* variants, int count, int planes, int64_t I, int64_t J, int64_t C, double split_us = 0) {
  Plan best{-1, 0, 0, 1};
  double best_us = 0;
  for (int v = 0; v < count; ++v) {
    const Variant& t = variants[v];
    if (t.planes != planes) continue;
    const int64_t tiles = ((I + t.bi - 1) / t.bi) * ((J + t.bj - 1) / t.bj), slots = 256 * t.per_cu;
    const int64_t stages = pad_to(C, kPad) / t.bk;
    const double rate = t.rate * 1e9 / slots;  // operations per us of one workgroup's slot
    auto rounds_us = [&](int64_t wgs, int64_t n) {  // wgs workgroups of n stages each
      const int64_t full = wgs / slots;
      const double r = (double)(wgs % slots) / slots;
      const double last = r == 0 ? 0 : t.per_cu == 1 ? t.partial : r * t.per_cu <= 1 ? 0.6 : 0.6 + 0.4 * r;
      return (full + last) * 2.0 * planes * t.bi * t.bj * n * t.bk / rate + t.round_us * (full + (r > 0));
    };
    auto consider = [&](int64_t full, int64_t ns, double us) {
      if (best.variant < 0 || us < best_us) best = {v, tiles, full, (int)ns}, best_us = us;
    };
    consider(tiles, 1, rounds_us(tiles, stages));
    for (int64_t want = 2; want <= 32 && stages / want >= 4; ++want) {
      const int64_t per = (stages + want - 1) / want, ns = (stages + per - 1) / per;  // no empty split
      if (ns != want) continue;
      for (const int64_t full : {(int64_t)0, tiles / slots * slots}) {
        const int64_t rest = tiles - full;
        if (rest == 0 || rest * ns > 4 * slots) continue;  // (no rest, or enough workgroups without so many parts)
        const double sums = 4.0 + split_us * ns + 8.0 * ns * rest * t.bi * t.bj / 8e6;
        consider(full, ns, (full ? rounds_us(full, stages) : 0) + rounds_us(rest * ns, per) + sums);
      }
    }
  }
  return best;
}

template <bool F16, int P, int TI, int TJ, int WI, int WJ, int BK, int WPE, int ST = 2>
hipError_t launch_tiles(const GradGemm& p, const Plan& pl, hipStream_t s) {
  constexpr int BI = 32 * TI * WI, BJ = 32 * TJ * WJ;
  const int ti = (p.I + BI - 1) / BI, tj = (p.J + BJ - 1) / BJ;
  const int64_t rest = pl.tiles - pl.full, grid = pad_to(pl.full, 8) + rest * pl.nsplit;
  if (grid > INT32_MAX) return hipErrorInvalidValue;
  hipLaunchKernelGGL((grad_tile_kernel<F16, P, TI, TJ, WI, WJ, BK, WPE, ST>), dim3((unsigned)grid), dim3(64 * WI * WJ), 0, s, p,
                     ti, tj);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || rest == 0) return e;
  hipLaunchKernelGGL(grad_reduce_kernel<F16>, dim3((unsigned)(rest * (BI * BJ / 2048))), dim3(256), 0, s, p, BI, BJ, ti, tj);
  return hipGetLastError();
}

constexpr int64_t align256(int64_t b) { return pad_to(b, 256); }

inline int64_t part_bytes_of(const Variant* variants, const Plan& pl) {
  return 4 * (pl.tiles - pl.full) * pl.nsplit * variants[pl.variant].bi * variants[pl.variant].bj;
}

// What launch_tiles needs to know of the plan and of the output.
inline void set_plan(GradGemm& p, const Plan& pl, const Variant* variants, int64_t C, float* parts) {
  p.stages = (int)(pad_to(C, kPad) / variants[pl.variant].bk);
  p.full = (int)pl.full;
  p.nsplit = pl.nsplit;
  p.parts = parts;
  const int osz = p.out_dtype == WFB_F32 ? 4 : 2;
  p.vec = (uintptr_t)p.out % 16 == 0 && (p.ldo * osz) % 16 == 0;
}

}  // namespace

}  // namespace wfb
