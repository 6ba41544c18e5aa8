// GQA attention over the int8 key/value cache (kv_i8.h): softmax(rope(q) . k * scale) v over the keys of a shared prefix
// and a sequence's own keys up to the query's position.
#include "kv_i8.h"

namespace wfb {

namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int kThreads = 256;
// Running maximum of a row that has met no key: finite, so that no difference is NaN, and not above any score.
constexpr float kNoMax = -3.40282347e38f;
constexpr float kLog2e = 1.4426950408889634f;

template <int DT>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float v) {
  if constexpr (DT == WFB_F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16_rne(v);
}

template <int DT>
__device__ __forceinline__ void store4(void* p, int64_t i, const float (&v)[4]) {
  if constexpr (DT == WFB_F32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    const bf16x2_t lo = __builtin_convertvector((f32x2_t){v[0], v[1]}, bf16x2_t);
    const bf16x2_t hi = __builtin_convertvector((f32x2_t){v[2], v[3]}, bf16x2_t);
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + i) =
        make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
  }
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = umax(v, (uint32_t)xor_lanes<32>((int)v));
  v = umax(v, (uint32_t)xor_lanes<16>((int)v));
  v = umax(v, (uint32_t)xor_lanes<8>((int)v));
  v = umax(v, (uint32_t)xor_lanes<4>((int)v));
  v = umax(v, (uint32_t)xor_lanes<2>((int)v));
  return umax(v, (uint32_t)xor_lanes<1>((int)v));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += xor_lanes_f32<32>(v);
  v += xor_lanes_f32<16>(v);
  v += xor_lanes_f32<8>(v);
  v += xor_lanes_f32<4>(v);
  v += xor_lanes_f32<2>(v);
  return v + xor_lanes_f32<1>(v);
}

// ---- plan ---------------------------------------------------------------------------------------

// How a call is cut: `own` workgroups along the sequences' own keys and `pre` along the prefix's, whose partial results
// (unnormalised output, running maximum, sum of weights) a last kernel joins; own = 1 without prefix needs none.
struct Plan {
  int own, pre;
  bool decode;    // one token per sequence: decode kernel, else the rows kernel
  bool pre_rows;  // the prefix by the rows kernel
  int waves;      // of a workgroup of prompt rows, 32 rows each
};

constexpr int kLive = 512;         // workgroups of four waves that fill the GPU: two per CU by their registers
constexpr int kColumns = 16;       // rows (token, query head) of a workgroup of decode_part
constexpr int kRowsWaves = 8;      // of a workgroup of prompt rows at most, 32 rows each
constexpr int kPrefixWaves = 4;    // of a workgroup of a decode step's rows against the prefix

int cut(int64_t groups, int64_t target, int64_t most) {
  const int64_t n = target / groups;
  return (int)(n > most ? (most < 1 ? 1 : most) : n < 1 ? 1 : n);
}

// keys: how many of their own the sequences of a prompt are expected to see (positions may be known on the device only).
// More keys never mean fewer splits, so cap gives the largest plan.  Times in us, of one call in a graph.
Plan make_plan(int dt, int64_t b, int64_t t, int64_t hq, int64_t hkv, int64_t d, int64_t cap, int64_t keys, int64_t npre,
               bool lengths) {
  const int64_t g = hq / hkv, pb = (npre + kKvBlock - 1) / kKvBlock, cb = cap / kKvBlock;
  Plan p{};
  p.decode = t == 1 && !lengths;
  if (p.decode) {
    // Splits of four blocks (one a wave) or more.  A cache of up to 1024 keys that needs no joining otherwise stays whole:
    // 3 heads of 64, 32-bit, whole against split at a quarter and at all of 512 keys 6.1, 7.8 against 8.6, 9.5; of 1024
    // 6.5, 10.1 against 9.3, 9.4; of 2048 7.7, 14.8 against 9.4, 10.0.
    p.own = npre == 0 && cb <= 16 ? 1 : cut(b * hkv, kLive, (cb + 3) / 4);
    // Splits of more than 64 blocks are halved, so that sequences of different lengths even out: 16 of 16384 to 32768 keys,
    // 8 heads of 128, 159.7 against 164.2; 16 of 32768 197.6, 198.3; 4 of 131071 195.9 against 192.3.
    if (cb / p.own > 64) p.own = cut(b * hkv, 2 * kLive, cb);
    if (npre > 0) {
      // The rows kernel reads a prefix once for 128 rows, where decode_part reads it for 16, but a block costs it three
      // times as much (32-bit: more), and converting it is lost on few rows.  decode_part against rows, c = columns * pb:
      // bf16, 8 heads of 128: 128 rows and 1024 keys (c 1024) 14.6, 19.7; 256 rows (2048) 23.9, 21.1; 64 rows and 4096 (2048)
      // 21.7, 21.2; 128 rows (4096) 22.9, 25.6; 128 rows and 16384 (16384) 40.1, 33.4; 512 rows (65536) 120.6, 69.4.
      // fp32 of 128: 256 rows and 8192 (16384) 45.2, 48.0; 512 rows and 4096 (16384) 52.5, 50.4; 1024 rows of 2 heads and
      // 16384 (32768) 65.9, 68.2; 256 rows of 8 (32768) 71.1 both; 512 rows and 8192 (32768) 78.9, 71.5; 16384 (65536) 123.9,
      // 116.2.  fp32 of 64: 256 rows and 4096 (8192) 24.2, 25.7; 8192 (16384) 30.3, 31.8; 16384 (32768) 44.2, 43.8; 512 rows
      // and 8192 (32768) 50.8, 42.0; 510 rows of 3 heads and 16384 (24576) 39.9, 38.4.
      const int64_t rows = b * g, columns = hkv * ((rows + kColumns - 1) / kColumns);
      p.pre_rows = rows > 32 && columns * pb > (dt == WFB_BF16 ? 1280 : d == 64 ? 16384 : 24576);
      if (p.pre_rows) p.pre = cut(hkv * ((rows + 32 * kPrefixWaves - 1) / (32 * kPrefixWaves)), 256, (pb + 3) / 4);
      else p.pre = cut(columns, kLive, (pb + 3) / 4);
    }
  } else {
    // Split where the GPU is not full and the keys are many: parts of every row go out and come back, 16 us for 65536 rows
    // of 128, what a workgroup needs for about 7 blocks.  8 heads of 128, whole against split: 512 tokens 26.9, 33.9, behind
    // 2048 keys 78.5, 51.2; 1024 tokens 41.2, 49.9, behind 2048 keys 91.9, 83.5.
    // Four waves, which convert a block for 128 rows instead of 256, where eight would leave rows or CUs empty: 8 heads of
    // 128, 4 query heads each, eight against four: 512 tokens 30.5, 27.0; 1024 46.1, 41.3; 2048 81.9, 74.5; 3000 114.5,
    // 112.3; 4096 182.8, 199.8; 16 tokens behind 4000 keys 27.6, 25.1; 8 x 48 behind 4000 shared keys, 5 heads, 46.7, 49.9.
    // (fp32 rows of 128 do not fit into the registers of four: 2 x 1587 tokens, 10 / 5 heads, 90.7, 101.7.)
    const int64_t rows = t * g, groups = b * hkv * ((rows + 32 * kRowsWaves - 1) / (32 * kRowsWaves));
    const int64_t blocks = pb + (keys + kKvBlock - 1) / kKvBlock;
    const int64_t n = cut(groups, 256, (blocks + 3) / 4);
    p.own = blocks * (n - 1) >= 9 * n ? (int)n : 1;
    p.waves = (rows <= 128 || (p.own == 1 && groups <= 384)) && (dt == WFB_BF16 || d == 64) ? 4 : kRowsWaves;
  }
  return p;
}

bool has_parts(const Plan& p) { return p.own > 1 || p.pre > 0; }

// Partials: unnormalised outputs [slots][rows][D], then maximum and sum [slots][rows]; row = (b * t + i) * hq + h.
struct Parts {
  float* o;
  float2* ml;
  int64_t rows;
};

Parts parts_of(const KvAttn& a, const Plan& p) {
  Parts r{nullptr, nullptr, (int64_t)a.b * a.t * a.hq};
  if (has_parts(p)) {
    r.o = a.ws;
    r.ml = reinterpret_cast<float2*>(a.ws + (int64_t)(p.own + p.pre) * r.rows * a.d);
  }
  return r;
}

// Blocks of 64 keys per split, in whole rounds of the four waves, when nb blocks are cut into at most n.
__device__ __forceinline__ int64_t split_blocks(int64_t nb, int n) { return ((nb + n - 1) / n + 3) / 4 * 4; }

// ---- decode: few rows -----------------------------------------------------------------------------

// Up to 16 rows (query heads of one kv head; behind a prefix also of several sequences) against the keys of a split, a
// 64-key block per wave at a time, straight from the cache into the matrix cores as they are stored:
//   S^T[key, row] = K Q^T        v_mfma_i32_16x16x64_i8, the query as NP signed base-256 digits of a fixed-point row
//   w = exp2(s - m) * v_scale    fp32, running maximum per row
//   O^T[d, row] = V^T W^T        the same instruction, w as NP digits of its block's largest in the row
// The products are exact; a block's sums of V^T W^T come to less than 2^31 (127 * 2^15 * 64 < 2^28) and are added up in fp32.
// The key that row R of score tile n stands for is chosen as 16 (R / 4) + 4 n + R % 4: a lane then holds 16 consecutive
// keys, the ones that it feeds into the second product.
// What bounds it: HBM where the cache is large (16 sequences of 16384 to 32768 keys, 8 heads of 128, 32 query heads, bf16:
// 0.7 GB in 143 us, 4.9 TB/s; one of 131071 keys and 5 heads 36 us, 4.8 TB/s), else the chain of one block's loads, products
// and exponentials (8 sequences of 1000 to 4096 keys: 44 MB in 15.2 us).  A wave's next block is fetched under the products
// of the one before; splits are sized so that two workgroups a CU are at work.  No conversion of codes and no LDS on the
// way: one key at a time in fp32, as the plain kernel had it, took 3.6 ms for the first of these.
template <int NP>
struct Digits;
template <>
struct Digits<2> {
  static constexpr float kMax = 127.0f * 256.0f;
};
template <>
struct Digits<3> {
  static constexpr float kMax = 127.0f * 65536.0f;
};

// Signed digits of four fixed-point numbers |x| <= Digits<NP>::kMax, packed, the most significant first: adding 0x80 to
// every lower byte carries a digit over 127 into the next one, and the byte less 128 is the digit.
template <int NP>
__device__ __forceinline__ void digits4(const int (&x)[4], uint32_t (&d)[NP]) {
  constexpr uint32_t bias = NP == 2 ? 0x80u : 0x8080u;
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = (uint32_t)x[i] + bias;
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    const uint32_t byte = NP - 1 - n;
    const uint32_t sel = byte | (byte + 4) << 8 | 0x0c0c0000u;  // byte of both sources, two zeros
    const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], sel), hi = __builtin_amdgcn_perm(u[3], u[2], sel);
    d[n] = (lo | hi << 16) ^ (n == 0 ? 0u : 0x80808080u);
  }
}

template <int NP, int D>
struct DecodeShared {
  uint8_t qd[NP][kColumns][D];  // the queries' digits
  float red[4][kColumns][D];    // the waves' outputs
  float mw[4][kColumns], lw[4][kColumns];
  float qscale[kColumns], snew[kColumns];
  float vnew[D];  // the new value as the cache holds it
};

template <int DT, int D, bool PREFIX>
__device__ __forceinline__ void decode_part(const KvAttn& a, const Parts& parts, int slot0, int nsplit, int kvh, int rowblock,
                                            int split, DecodeShared<DT == WFB_F32 ? 3 : 2, D>& sh) {
  constexpr int NP = DT == WFB_F32 ? 3 : 2;
  constexpr int HD = D / 2, KS = D / 64, DTL = D / 16, E = D / 64;
  constexpr float QM = Digits<NP>::kMax;
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int g = a.hq / a.hkv;
  const int grp = lane >> 4, col = lane & 15;
  // rows of this workgroup: the heads of one sequence, or the next 16 of all sequences' (sequence, head) pairs
  const int b0 = PREFIX ? 0 : rowblock, r0 = PREFIX ? rowblock * kColumns : 0;
  const int nrows = PREFIX ? (a.b * g - r0 < kColumns ? a.b * g - r0 : kColumns) : g;
  int64_t pos = 0;
  int n1 = 1;
  if constexpr (!PREFIX) {
    if (!kv_span(a.span, b0, pos, n1)) {  // uniform: the rows are flagged, here or by the joining kernel
      if (!parts.o)
        for (int i = t; i < g * D; i += kThreads)
          store_elem<DT>(a.out, (int64_t)b0 * a.ldo + (int64_t)kvh * g * D + i, __builtin_nanf(""));
      return;
    }
  }
  const int64_t keys = PREFIX ? a.npre : pos;  // read from the cache
  const int64_t nb = (keys + kKvBlock - 1) / kKvBlock, per = split_blocks(nb, nsplit);
  const int64_t kb0 = split * per, kb1 = kb0 + per < nb ? kb0 + per : nb;
  if (split > 0 && kb0 >= nb) return;  // (split 0 of a sequence without older keys takes the new one)
  const bool owns_new = !PREFIX && kb1 == nb;

  const wfb_kv_i8& c = PREFIX ? a.pre : a.own;
  const int64_t base = PREFIX ? kvh : (int64_t)b0 * a.hkv + kvh;
  const int8_t* kp = c.k + base * c.cap * D;
  const int8_t* vp = c.v + base * c.cap * D;
  // codes behind the last key are met with weights of zero; scales there read as zeros
  const buf_t ksb = make_buf(c.k_scale + base * c.cap, (uint32_t)(keys * 4));
  const buf_t vsb = make_buf(c.v_scale + base * c.cap, (uint32_t)(keys * 4));

  v4i kf[4][KS], vf[DTL], sk[4], sv[4];
  auto load_k = [&](int64_t kb) {
    const buf_t p = make_buf(kp + kb * kKvBlock * D, kKvBlock * D);
    const int off = (16 * (col >> 2) + (col & 3)) * D + 16 * grp;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[n][s] = buf_load16(p, off + 4 * n * D + 64 * s);
  };
  auto load_v = [&](int64_t kb) {
    const buf_t p = make_buf(vp + kb * kKvBlock * D, kKvBlock * D);
    const int off = col * kKvBlock + 16 * grp;
#pragma unroll
    for (int d = 0; d < DTL; ++d) vf[d] = buf_load16(p, off + 16 * d * kKvBlock);
  };
  auto load_s = [&](int64_t kb) {
    const uint32_t off = (uint32_t)(kb * kKvBlock + 16 * grp) * 4;
#pragma unroll
    for (int n = 0; n < 4; ++n) sk[n] = buf_load16(ksb, off + 16 * n);
#pragma unroll
    for (int n = 0; n < 4; ++n) sv[n] = buf_load16(vsb, off + 16 * n);
  };
  // ---- a wave's rows w, w + 4, .. and the new key, elements lane and lane + 64, and the first block's loads: these come
  // last, since loads complete in the order of their issue
  float x[4][E], xc[4], xs[4], kn[E], vn[E];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = w + 4 * i;  // uniform
#pragma unroll
    for (int e = 0; e < E; ++e) x[i][e] = 0.0f;
    xc[i] = 1.0f;
    xs[i] = 0.0f;
    if (r >= nrows) continue;
    const int sb = PREFIX ? (r0 + r) / g : b0, h = kvh * g + (PREFIX ? (r0 + r) % g : r);
    int64_t p = pos;
    if constexpr (PREFIX)
      if (!kv_span(a.span, sb, p, n1)) continue;  // (its result is not used)
    const int64_t off = (int64_t)sb * a.ldq + (int64_t)h * D;
#pragma unroll
    for (int e = 0; e < E; ++e) x[i][e] = load_elem<DT>(a.q, off + lane + 64 * e);
    if (a.rc) {
      xc[i] = a.rc[(p + a.npre) * HD + lane % HD];
      xs[i] = a.rs[(p + a.npre) * HD + lane % HD];
    }
  }
  float kc = 1.0f, ks = 0.0f;
  if (owns_new) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      kn[e] = load_elem<DT>(a.kn, (int64_t)b0 * a.ldk + (int64_t)kvh * D + lane + 64 * e);
      vn[e] = load_elem<DT>(a.vn, (int64_t)b0 * a.ldv + (int64_t)kvh * D + lane + 64 * e);
    }
    if (a.rc) {
      kc = a.rc[(pos + a.npre) * HD + lane % HD];
      ks = a.rs[(pos + a.npre) * HD + lane % HD];
    }
  }
  int64_t kb = kb0 + w;
  if (kb < kb1) {
    load_k(kb);
    load_s(kb);
    load_v(kb);
  }
  auto turn = [&](float (&y)[E], float cs, float sn) {  // (tables of ones and zeros where there are none)
    if constexpr (E == 2) {
      const float y1 = __fsub_rn(__fmul_rn(y[0], cs), __fmul_rn(y[1], sn));
      y[1] = __fadd_rn(__fmul_rn(y[1], cs), __fmul_rn(y[0], sn));
      y[0] = y1;
    } else {
      const float other = xor_lanes_f32<32>(y[0]), p = __fmul_rn(y[0], cs), q = __fmul_rn(other, sn);
      y[0] = lane < 32 ? __fsub_rn(p, q) : __fadd_rn(p, q);
    }
  };
  auto largest = [&](const float (&y)[E]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) m = umax(m, __float_as_uint(y[e]) & 0x7fffffffu);
    return wave_umax(m);
  };
  if (owns_new) {  // every wave forms the key that the cache holds, wave 0 writes it, wave 1 the value
    if (a.rc) turn(kn, kc, ks);
    float scale, inv;
    kv_scale(largest(kn), scale, inv);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int q = kv_code(kn[e], inv);
      if (w == 0) a.own.k[(base * c.cap + pos) * D + lane + 64 * e] = (int8_t)q;
      kn[e] = (float)q * scale;
    }
    if (w == 0 && lane == 0) a.own.k_scale[base * c.cap + pos] = scale;
    if (w == 1) {
      kv_scale(largest(vn), scale, inv);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int q = kv_code(vn[e], inv);
        a.own.v[(base * c.cap + pos / kKvBlock * kKvBlock) * D + (int64_t)(lane + 64 * e) * kKvBlock + pos % kKvBlock] =
            (int8_t)q;
        sh.vnew[lane + 64 * e] = (float)q * scale;
      }
      if (lane == 0) a.own.v_scale[base * c.cap + pos] = scale;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = w + 4 * i;
    if (i > 0 && r >= (nrows + 3) / 4 * 4) {  // uniform: rows of zeros
#pragma unroll
      for (int n = 0; n < NP; ++n)
#pragma unroll
        for (int e = 0; e < E; ++e) sh.qd[n][r][lane + 64 * e] = 0;
      if (lane == 0) sh.qscale[r] = 0.0f;
      continue;
    }
    if (a.rc) turn(x[i], xc[i], xs[i]);
    const uint32_t m = largest(x[i]);
    const float mf = __uint_as_float(m);
    const bool some = m < 0x7f800000u && mf >= kKvTiny;
    const float inv = some ? (a.scale < 0.0f ? -QM : QM) / mf : 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int q = some ? (int)__builtin_rintf(x[i][e] * inv) : 0;
      const uint32_t u = (uint32_t)q + (NP == 2 ? 0x80u : 0x8080u);
#pragma unroll
      for (int n = 0; n < NP; ++n)
        sh.qd[n][r][lane + 64 * e] = (uint8_t)((u >> 8 * (NP - 1 - n)) ^ (n == 0 ? 0u : 0x80u));
    }
    if (lane == 0)  // one step of the digits in units of the exponent of two; NaN for a row with one
      sh.qscale[r] = m >= 0x7f800000u ? __builtin_nanf("") : some ? mf * (1.0f / QM) * (fabsf(a.scale) * kLog2e) : 0.0f;
    if (owns_new) {
      float p = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) p += x[i][e] * kn[e];
      p = wave_sum(p);
      if (lane == 0) sh.snew[r] = p * (a.scale * kLog2e);
    }
  }
  __syncthreads();
  v4i qf[NP][KS];
#pragma unroll
  for (int n = 0; n < NP; ++n)
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[n][s] = *reinterpret_cast<const v4i*>(&sh.qd[n][col][64 * s + 16 * grp]);
  const float cq = sh.qscale[col];

  float o[DTL][4];
#pragma unroll
  for (int d = 0; d < DTL; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[d][i] = 0.0f;
  float m_run = kNoMax, l_run = 0.0f;

  for (; kb < kb1; kb += 4) {
    const bool more = kb + 4 < kb1;
    float s[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      v4i acc = {0, 0, 0, 0}, low = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < KS; ++k) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[n][k], qf[0][k], acc, 0, 0, 0);
      acc <<= 8;
#pragma unroll
      for (int k = 0; k < KS; ++k) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[n][k], qf[1][k], acc, 0, 0, 0);
      if constexpr (NP == 3) {
#pragma unroll
        for (int k = 0; k < KS; ++k) low = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[n][k], qf[2][k], low, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[n][i] = (NP == 3 ? __builtin_fmaf((float)acc[i], 256.0f, (float)low[i]) : (float)acc[i]) *
                  (cq * __int_as_float(sk[n][i]));
    }
    if (more) load_k(kb + 4);
    const int left = (int)(keys - kb * kKvBlock);  // keys of this block that there are
    if (left < kKvBlock) {
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * grp + 4 * n + i >= left) s[n][i] = -__builtin_inff();
    }
    float mx = s[0][0];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[n][i]);
    mx = fmaxf(mx, xor_lanes_f32<16>(mx));
    mx = fmaxf(mx, xor_lanes_f32<32>(mx));
    const float m_new = fmaxf(m_run, mx), alpha = __builtin_amdgcn_exp2f(m_run - m_new);
    m_run = m_new;
    float ps = 0.0f;
    uint32_t wm = 0;  // the largest weight, as bits: a NaN is larger than any number
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(s[n][i] - m_new);
        ps += p;
        s[n][i] = p * __int_as_float(sv[n][i]);
        wm = umax(wm, __float_as_uint(s[n][i]));
      }
    if (more) load_s(kb + 4);
    l_run = l_run * alpha + ps;
    wm = umax(wm, (uint32_t)xor_lanes<16>((int)wm));
    wm = umax(wm, (uint32_t)xor_lanes<32>((int)wm));
    // step of the weights' digits; not below 2^-120, so that its inverse is finite (and left NaN)
    float step = __uint_as_float(wm) * (1.0f / QM);
    step = step < 0x1p-120f ? 0x1p-120f : step;
    const float inv = __builtin_amdgcn_rcpf(step);
    v4i pf[NP];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      int x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (int)__builtin_rintf(s[n][i] * inv);
      uint32_t dg[NP];
      digits4<NP>(x, dg);
#pragma unroll
      for (int k = 0; k < NP; ++k) pf[k][n] = (int)dg[k];
    }
#pragma unroll
    for (int d = 0; d < DTL; ++d) {
      v4i acc = {0, 0, 0, 0}, low = {0, 0, 0, 0};
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[d], pf[0], acc, 0, 0, 0);
      acc <<= 8;
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[d], pf[1], acc, 0, 0, 0);
      if constexpr (NP == 3) low = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[d], pf[2], low, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = NP == 3 ? __builtin_fmaf((float)acc[i], 256.0f, (float)low[i]) : (float)acc[i];
        o[d][i] = __builtin_fmaf(o[d][i], alpha, x * step);
      }
    }
    if (more) load_v(kb + 4);
  }

  l_run += xor_lanes_f32<16>(l_run);
  l_run += xor_lanes_f32<32>(l_run);
  if (grp == 0) {
    sh.mw[w][col] = m_run;
    sh.lw[w][col] = l_run;
  }
  if (col < nrows) {
#pragma unroll
    for (int d = 0; d < DTL; ++d)
      *reinterpret_cast<float4*>(&sh.red[w][col][16 * d + 4 * grp]) = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
  }
  __syncthreads();
  // the four waves and the new key, four elements of a row per thread
  for (int i = t; i < nrows * (D / 4); i += kThreads) {
    const int r = i / (D / 4), j = 4 * (i % (D / 4));
    float m = fmaxf(fmaxf(sh.mw[0][r], sh.mw[1][r]), fmaxf(sh.mw[2][r], sh.mw[3][r]));
    if (owns_new) m = fmaxf(m, sh.snew[r]);
    float l = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float e = __builtin_amdgcn_exp2f(sh.mw[x][r] - m);
      const float4 f = *reinterpret_cast<const float4*>(&sh.red[x][r][j]);
      l += sh.lw[x][r] * e;
      v[0] += f.x * e;
      v[1] += f.y * e;
      v[2] += f.z * e;
      v[3] += f.w * e;
    }
    if (owns_new) {
      const float e = __builtin_amdgcn_exp2f(sh.snew[r] - m);
      l += e;
#pragma unroll
      for (int x = 0; x < 4; ++x) v[x] += e * sh.vnew[j + x];
    }
    const int sb = PREFIX ? (r0 + r) / g : b0, h = kvh * g + (PREFIX ? (r0 + r) % g : r);
    if (parts.o) {
      const int64_t row = (int64_t)(slot0 + split) * parts.rows + (int64_t)sb * a.hq + h;
      *reinterpret_cast<float4*>(parts.o + row * D + j) = make_float4(v[0], v[1], v[2], v[3]);
      if (j == 0) parts.ml[row] = make_float2(m, l);
    } else {
#pragma unroll
      for (int x = 0; x < 4; ++x) v[x] /= l;
      store4<DT>(a.out, (int64_t)sb * a.ldo + (int64_t)h * D + j, v);
    }
  }
}

// ---- prompt chunks, and a prefix that many rows share ------------------------------------------------

// Four codes as fp16, exactly: a code plus 128 in the low byte of 0x64xx is 1024 + 128 + code.
__device__ __forceinline__ void codes_to_f16(int codes, int& f0, int& f1) {
  const uint32_t u = (uint32_t)codes ^ 0x80808080u;
  const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);  // bytes u0, 64, u1, 64
  const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
  const f16x2_t k = {(_Float16)1152.0f, (_Float16)1152.0f};
  f0 = __builtin_bit_cast(int, __builtin_bit_cast(f16x2_t, lo) - k);
  f1 = __builtin_bit_cast(int, __builtin_bit_cast(f16x2_t, hi) - k);
}

// Two numbers as packed fp16: one part, or two (x = hi + lo to 22 bits).  The packed pair is pinned before lo is formed: the
// compiler may fold the product behind x into one of two conversions only, and the two round differently.
template <int NP>
__device__ __forceinline__ void f16_parts(float x0, float x1, uint32_t (&part)[NP]) {
  const f16x2_t hi = {(_Float16)x0, (_Float16)x1};
  uint32_t h = __builtin_bit_cast(uint32_t, hi);
  if constexpr (NP == 2) {
    asm("" : "+v"(h));
    const f16x2_t b = __builtin_bit_cast(f16x2_t, h);
    const f16x2_t lo = {(_Float16)(x0 - (float)b[0]), (_Float16)(x1 - (float)b[1])};
    part[NP - 1] = __builtin_bit_cast(uint32_t, lo);
  }
  part[0] = h;
}

// Rows r of one kv head (row r: token r / G, query head r % G), 32 per wave of W, against blocks of 64 keys that the
// workgroup converts to fp16 (exactly) into LDS.  PREFIX: the rows of all sequences of a decode step against the
// shared prefix; else the prefix first, if there is one, then the sequence's own keys, causal.
//   S^T[key, row] = K Q^T         v_mfma_f32_32x32x16_f16; q in fp16 of its row's largest (fp32 rows: two parts)
//   p = exp2(s k_scale c - m)     fp32, a reference m that follows the row's maximum from below
//   O^T[d, row] += V^T W^T        w = p v_scale / (reference of the scales) in fp16 (fp32 rows: two parts)
// As in the decode kernel the key of a score tile's row is chosen so that a lane holds the keys that it feeds into the
// second product, 8 consecutive ones per step.
// What bounds it: nothing alone.  4096 tokens, 32 / 8 heads of 128, bf16: 137 GFLOP in 188 to 190 us (0.73 PFLOP/s); the
// matrix cores are busy 34% of the cycles, vector instructions 44%, LDS about half, since a product of 32 x 32 x 16 reads 16
// bytes a lane of it; two waves a SIMD (by their registers) leave the rest to latency.  A block costs 256 rows 2.0 to 2.8 us.
// Tried without gain: the two waves of a SIMD half a block apart (197 against 187 us), 64 rows a wave and one wave a SIMD
// (331: 100 spilled registers), the exponentials a block ahead of their products (5% slower).
template <int D>
struct RowsShared {
  uint16_t tile[2][2][kKvBlock * D];  // [buffer][keys, values]
  // scales of a block's keys and values and of the two behind it; svs: as fp16 if kScaled
  float sks[3][kKvBlock], svs[3][kKvBlock];
  float vref_s[3];
};

template <int DT, int D, int W, bool PREFIX>
__device__ __forceinline__ void rows_part(const KvAttn& a, const Parts& parts, int slot0, int nsplit, int block_id,
                                          RowsShared<D>& sh) {
  constexpr int NP = DT == WFB_F32 ? 2 : 1;
  constexpr int kRows = 32 * W;
  // With one part the values' scales are multiplied into their codes as these become fp16 (two roundings to 11 bits of a
  // value, like that of p, an eighth of the output's); with two they stay factors of the weights.  The keys' scales are
  // factors of the scores in both: a score may be large, and 11 bits of it too few.
  constexpr bool kScaled = NP == 1;
  constexpr int HD = D / 2, KS = D / 16, DTL = D / 32;
  // The weights' reference m_ref is set kDown below the row's maximum and moves once that is more than kSlack above it, so
  // weights reach 2^kSlack; a value scale is at most half its reference, in every block.  fp16 ends at 65504 and holds 11
  // bits down to 2^-14.  One part: weights of 2^10 to 2^15 at the maximum have 11 bits down to 2^-24 of the row's largest
  // (16.6 nats; with kDown = 0, kSlack = 8 only to 2^-14, and equal keys 16 nats below one whose value is nothing came out
  // 18% off; a prompt of 4096 tokens takes 189 us with kDown = 0 to 12, 193 with 14, a step of 64 sequences behind 8192 keys
  // 39.3 with 0, 40.1 with 10),
  // and values stay below 127 kUp / 2 < 2^14.  Two parts: weights times kUp / 2 reach 2^15, which keeps the lower part of
  // weights down to 2^-16 of the row's largest out of the subnormal numbers; below, they are exact to 2^-38 of it.
  constexpr float kDown = NP == 1 ? 10.0f : 0.0f, kSlack = NP == 1 ? 15.0f : 1.0f, kUp = NP == 1 ? 0x1p8f : 0x1p15f;
  constexpr int kRingK = 4, kRingV = 4;  // fragments read ahead of their products
  constexpr int CK = D / 16;             // pieces of 16 codes of a key
  constexpr int KP = kKvBlock * CK;      // of a block's keys; as many of its values
  constexpr int PT = 2 * KP / (64 * W);  // per thread
  static_assert(PT * 64 * W == 2 * KP && KP % 64 == 0, "whole waves take keys or values");
  static_assert(KP % (64 * W) == 0 || D == kKvBlock, "a round of keys and values needs rows of one length");
  auto& tile = sh.tile;
  auto& sks = sh.sks;
  auto& svs = sh.svs;
  auto& vref_s = sh.vref_s;

  const int g = a.hq / a.hkv;
  const int nhb = PREFIX ? a.hkv : a.hkv * a.b;
  const int64_t R = PREFIX ? (int64_t)a.b * g : (int64_t)a.t * g;
  const int nrb = (int)((R + kRows - 1) / kRows);
  // the heads' workgroups are nhb apart, so an XCD's L2 holds few heads; the longest rows (the last) come first
  const int hb = block_id % nhb, rest = block_id / nhb;
  const int split = rest % nsplit, rb = nrb - 1 - rest / nsplit;
  const int kvh = hb % a.hkv, b = hb / a.hkv;
  const int t = threadIdx.x, lane = t & 63;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int col = lane & 31, grp = lane >> 5;
  const int64_t r = (int64_t)rb * kRows + 32 * w + col;
  const int tok = (int)(r / g), h = kvh * g + (int)(r % g);

  int64_t first = 0;
  int n = 0;
  bool fits = true;
  bool valid = r < R;
  if constexpr (PREFIX) {
    valid = valid && kv_span(a.span, tok, first, n);
  } else {
    fits = kv_span(a.span, b, first, n);
    valid = valid && fits && tok < n;
  }
  const int64_t pos = PREFIX ? first : first + tok;
  const int64_t rw = (int64_t)rb * kRows + 32 * w;  // the wave's first row and (not PREFIX) its position
  const int64_t pos_low = first + rw / g;
  const int64_t qrow = PREFIX ? tok : (int64_t)b * a.t + tok;
  int64_t own = 0;  // own keys that the workgroup's last row sees
  if constexpr (!PREFIX) {
    const int64_t tok0 = (int64_t)rb * kRows / g;
    if (!fits || tok0 >= n) {  // uniform: no row here
      if (!parts.o && r < R) {
        const float v = fits ? 0.0f : __builtin_nanf("");
        const float v4[4] = {v, v, v, v};
        for (int j = 4 * grp; j < D; j += 8) store4<DT>(a.out, qrow * a.ldo + (int64_t)h * D + j, v4);
      }
      return;
    }
    const int64_t tok1 = ((int64_t)(rb + 1) * kRows + g - 1) / g;  // past the last row's token
    own = first + (tok1 < n ? tok1 : n);
  }
  // (blocks in 32 bits: a comparison of 64 is a vector instruction, and what hangs on it no longer uniform to the compiler)
  const int pb = (int)((a.npre + kKvBlock - 1) / kKvBlock), nb = pb + (int)((own + kKvBlock - 1) / kKvBlock);
  const int per = (nb + nsplit - 1) / nsplit;
  const int kb0 = split * per, kb1 = kb0 + per < nb ? kb0 + per : nb;

  // ---- staging: K row-major [key][D], V as it is [element][64 keys], 16-byte chunks at chunk ^ (row's swizzle) so that
  // 16 lanes reading one chunk of 16 rows meet 16 different bank groups
  auto kswz = [](int key) { return D == 128 ? key & 15 : (key >> 1) & 7; };
  auto vswz = [](int d) { return (d >> 1) & 7; };
  v4i raw[2][PT] = {};  // codes of the next block and of the one behind it
  const int64_t pre_at = kvh * a.pre.cap, own_at = ((int64_t)b * a.hkv + kvh) * a.own.cap;
  const int pre_tail = (int)(a.npre - (int64_t)(pb - 1) * kKvBlock);  // keys of the last blocks
  const int own_tail = (int)(own - (int64_t)(nb - pb - 1) * kKvBlock);
  // The first key of a block in its cache.  (Members are chosen one by one: a choice between the two structs would have to
  // be read through a pointer, in every block.)
  auto first_key = [&](int kb) { return kb < pb ? pre_at + (int64_t)kb * kKvBlock : own_at + (int64_t)(kb - pb) * kKvBlock; };
  auto fetch_codes = [&](int kb, int set) {
    const int64_t at = first_key(kb) * D;
    const buf_t kb_ = make_buf((kb < pb ? a.pre.k : a.own.k) + at, kKvBlock * D);
    const buf_t vb_ = make_buf((kb < pb ? a.pre.v : a.own.v) + at, kKvBlock * D);
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int p0 = 64 * (w + i * W);  // uniform
      const bool isk = 64 * W * (i + 1) <= KP || (64 * W * i < KP && p0 < KP);
      raw[set][i] = buf_load16(isk ? kb_ : vb_, 16 * ((isk ? p0 : p0 - KP) + lane));
    }
  };
  float sk = 0.0f, sv = 0.0f;  // the scales of key `lane`, zeros behind the last key; waves 0 and 1 stage them
  auto fetch_scales = [&](int kb) {
    const int64_t at = first_key(kb);
    const uint32_t bytes = 4 * (kb == pb - 1 ? pre_tail : kb == nb - 1 ? own_tail : kKvBlock);
    const buf_t ks = make_buf((kb < pb ? a.pre.k_scale : a.own.k_scale) + at, bytes);
    const buf_t vs = make_buf((kb < pb ? a.pre.v_scale : a.own.v_scale) + at, bytes);
    sk = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(ks, 4 * lane, 0, 0));
    sv = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(vs, 4 * lane, 0, 0));
  };
  float sk1 = 0.0f, sv1 = 0.0f;
  if (kb0 < kb1) {  // under way while the queries are formed
    fetch_scales(kb0 + 1 < kb1 ? kb0 + 1 : kb0);
    sk1 = sk;
    sv1 = sv;
    fetch_scales(kb0);
    fetch_codes(kb0, 0);
    fetch_codes(kb0 + 1 < kb1 ? kb0 + 1 : kb0, 1);
  }

  // ---- the row's query in fp16 of its largest: lane holds elements 16 s + 8 grp .. + 7
  v4i qf[NP][KS];
  float cq;
  {
    float x[KS][8];
    uint32_t m = 0;
    if (valid) {
#pragma unroll
      for (int s = 0; s < KS; ++s) load8<DT>(a.q, qrow * a.ldq + (int64_t)h * D + 16 * s + 8 * grp, x[s]);
      if (a.rc) {
#pragma unroll
        for (int s = 0; s < KS / 2; ++s) {
          float cs[8], sn[8];
          load8<WFB_F32>(a.rc, (pos + a.npre) * HD + 16 * s + 8 * grp, cs);
          load8<WFB_F32>(a.rs, (pos + a.npre) * HD + 16 * s + 8 * grp, sn);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x1 = x[s][j], x2 = x[s + KS / 2][j];
            x[s][j] = __fsub_rn(__fmul_rn(x1, cs[j]), __fmul_rn(x2, sn[j]));
            x[s + KS / 2][j] = __fadd_rn(__fmul_rn(x2, cs[j]), __fmul_rn(x1, sn[j]));
          }
        }
      }
    } else {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[s][j] = 0.0f;
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = umax(m, __float_as_uint(x[s][j]) & 0x7fffffffu);
    m = umax(m, (uint32_t)xor_lanes<32>((int)m));
    // by a power of two to [2^14, 2^15): exact, the small elements far from fp16's subnormal numbers
    const bool some = m < 0x7f800000u && __uint_as_float(m) >= kKvTiny;
    const int e = (int)(m >> 23) - 127;
    const float up = some ? __uint_as_float((uint32_t)(127 + 14 - e) << 23) : 0.0f;
    const float down = some ? __uint_as_float((uint32_t)(127 - 14 + e) << 23) : 0.0f;
    const float sign = a.scale < 0.0f ? -up : up;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float y0 = some ? x[s][j] * sign : 0.0f, y1 = some ? x[s][j + 1] * sign : 0.0f;
        uint32_t part[NP];
        f16_parts<NP>(y0, y1, part);
#pragma unroll
        for (int p = 0; p < NP; ++p) qf[p][s][j / 2] = (int)part[p];
      }
    // not below the smallest normal number: a masked score's -inf must not meet a zero
    cq = fmaxf(down * (fabsf(a.scale) * kLog2e), 0x1p-126f);
    if (m >= 0x7f800000u) cq = __builtin_nanf("");
  }

  f32x16_t o[DTL];
#pragma unroll
  for (int d = 0; d < DTL; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  float m_ref = kNoMax, l_run = 0.0f, vref = 0x1p-100f;
  // A weight's exponent is s cq - m_ref with one rounding, where m_ref comes from a rounded product: the two may differ by
  // half a unit of m_ref's last place, which is nothing below kFar and, far above it, whole powers of two.  A wave with such a
  // reference multiplies first (and takes the maximum itself, since one kDown below it need not be a number).
  constexpr float kFar = 0x1p20f;
  bool far = false;

  float ref = 0x1p-100f;  // (wave 1) reference of the value scales so far
  auto stage_scales = [&](int slot) {
    // a value row that is not finite makes NaN of its key's scores, which a mask can take away, and counts as zeros
    if (w == 0) {
      sks[slot][lane] = sv != sv ? sv : sk;
    } else if (w == 1) {
      const float x = fmaxf(sv, 0.0f);
      float mx = x;
      mx = fmaxf(mx, xor_lanes_f32<32>(mx));
      mx = fmaxf(mx, xor_lanes_f32<16>(mx));
      mx = fmaxf(mx, xor_lanes_f32<8>(mx));
      mx = fmaxf(mx, xor_lanes_f32<4>(mx));
      mx = fmaxf(mx, xor_lanes_f32<2>(mx));
      mx = fmaxf(mx, xor_lanes_f32<1>(mx));
      if (2.0f * mx > ref)  // twice the power of two at or above it: growth up to that power costs nothing
        ref = __uint_as_float(((__float_as_uint(mx) + 0x7fffffu) & 0x7f800000u) + 0x800000u);
      const float y = x * (kUp * __uint_as_float(0x7f000000u - __float_as_uint(ref)));
      if constexpr (kScaled) reinterpret_cast<_Float16*>(svs[slot])[lane] = (_Float16)y;
      else svs[slot][lane] = y;
      if (lane == 0) vref_s[slot] = ref;
    }
  };
  // pieces of 16 codes: whole waves, and but for D = 64 with 8 waves whole rounds, take keys or values; there the row
  // formulas of the two agree
  auto piece = [&](int i, bool& isk, int& row, int& c) {
    const int p0 = 64 * (w + i * W);
    isk = 64 * W * (i + 1) <= KP || (64 * W * i < KP && p0 < KP);
    const int p = (isk ? p0 : p0 - KP) + lane, per = 64 * W * (i + 1) <= KP ? CK : 4;
    row = p / per;
    c = p % per;
  };
  v4i half[2];
  uint32_t factor[8];
  auto read_factors = [&](int i, int slot) {  // of piece i
    if constexpr (kScaled) {
      if (64 * W * (i + 1) <= KP) return;
      bool isk;
      int row, c;
      piece(i, isk, row, c);
      const v4i f0 = *reinterpret_cast<const v4i*>(&svs[slot][8 * c]);
      const v4i f1 = *reinterpret_cast<const v4i*>(&svs[slot][8 * c + 4]);
#pragma unroll
      for (int x = 0; x < 8; ++x) factor[x] = isk ? 0x3c003c00u : (uint32_t)(x < 4 ? f0[x] : f1[x - 4]);  // (ones)
    }
  };
  auto convert = [&](int i, int set) {  // word i of the thread's codes
    int f[2];
    codes_to_f16(raw[set][i / 4][i % 4], f[0], f[1]);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (kScaled && 64 * W * (i / 4 + 1) > KP)
        f[x] = __builtin_bit_cast(
            int, __builtin_bit_cast(f16x2_t, f[x]) * __builtin_bit_cast(f16x2_t, factor[2 * (i % 4) + x]));
      half[i % 4 / 2][2 * (i % 2) + x] = f[x];
    }
  };
  auto stage_codes = [&](int i, int buf) {  // piece i
    bool isk;
    int row, c;
    piece(i, isk, row, c);
    const bool krow = 64 * W * (i + 1) <= KP;
    const int x = krow ? kswz(row) : vswz(row);
    uint16_t* dst = &tile[buf][isk ? 0 : 1][row * (krow ? D : kKvBlock)];
    *reinterpret_cast<v4i*>(dst + 8 * ((2 * c) ^ x)) = half[0];
    *reinterpret_cast<v4i*>(dst + 8 * ((2 * c + 1) ^ x)) = half[1];
  };

  const int key = 16 * (col >> 4) + 8 * ((col >> 2) & 1) + 4 * ((col >> 3) & 1) + (col & 3);
  const int ka = key * D, kx = kswz(key), va = col * kKvBlock, vx = vswz(col);  // (a tile's 32 rows repeat the swizzle)
  // Block kb, in buffer buf and scale slot `slot`.  Under the first products the next block's codes, fetched during the
  // block before, become fp16 and then go to the other buffer; the scales of the one behind it go to the next slot but one.
  auto block = [&](int kb, int buf, int slot) {
    const int slot1 = slot == 2 ? 0 : slot + 1, slot2 = slot1 == 2 ? 0 : slot1 + 1;
    const uint16_t* ks = tile[buf][0];
    const uint16_t* vs = tile[buf][1];
    fetch_codes(kb + 2 < kb1 ? kb + 2 : kb1 - 1, buf);  // (always: behind a branch every wait would be for all loads)
    read_factors(0, slot1);
    const float vnew = vref_s[slot];
    if (vnew != vref) {  // uniform
      const float f = vref / vnew;
      vref = vnew;
#pragma unroll
      for (int d = 0; d < DTL; ++d) o[d] *= f;
    }
    // S^T, fragments kRingK steps ahead of their products; row R = 8 a + 4 e + i of a tile stands for key 16 (a / 2) + 8 e +
    // 4 (a % 2) + i
    f32x16_t s[2];
#pragma unroll
    for (int nb2 = 0; nb2 < 2; ++nb2)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[nb2][i] = 0.0f;
    {
      v4i f[kRingK];
      auto read_k = [&](int i) {
        f[i % kRingK] = *reinterpret_cast<const v4i*>(&ks[32 * D * (i & 1) + ka + 8 * ((2 * (i >> 1) + grp) ^ kx)]);
      };
#pragma unroll
      for (int i = 0; i < kRingK; ++i) read_k(i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) {  // in this order: a product, a read ahead, a part of the conversion
#pragma unroll
        for (int p = 0; p < NP; ++p)
          s[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, f[i % kRingK]),
                                                            __builtin_bit_cast(f16x8_t, qf[p][i >> 1]), s[i & 1], 0, 0, 0);
        if (i + kRingK < 2 * KS) read_k(i + kRingK);
        // word x of the codes behind step (x + 1) 2 KS / (4 PT) - 1, the last of a piece with the piece's way to the tile
        // (behind the last block: of no meaning, and never read)
#pragma unroll
        for (int x = 0; x < 4 * PT; ++x)
          if (i == (x + 1) * 2 * KS / (4 * PT) - 1) {
            convert(x, buf ^ 1);
            if (x % 4 == 3) {
              stage_codes(x / 4, buf ^ 1);
              if (x / 4 + 1 < PT) read_factors(x / 4 + 1, slot1);
            }
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    stage_scales(slot2);
    fetch_scales(kb + 3 < kb1 ? kb + 3 : kb1 - 1);
    // register 8 c + j of tile nb2 holds key 32 nb2 + 16 c + 8 grp + j
    float bmax = -__builtin_inff();
#pragma unroll
    for (int nb2 = 0; nb2 < 2; ++nb2)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const float4 f = *reinterpret_cast<const float4*>(&sks[slot][32 * nb2 + 16 * (i / 8) + 8 * grp + i % 8]);
        s[nb2][i] *= f.x;
        s[nb2][i + 1] *= f.y;
        s[nb2][i + 2] *= f.z;
        s[nb2][i + 3] *= f.w;
      }
    // keys of the block that the row sees, and the wave's first one, if not all of them
    const int64_t k0 = (int64_t)(kb - pb) * kKvBlock;
    auto sees = [&](int64_t p) { return p + 1 - k0 > kKvBlock ? kKvBlock : (int)(p + 1 - k0); };
    const int low = kb < pb - 1 ? kKvBlock : kb == pb - 1 ? pre_tail : sees(pos_low);
    if (low < kKvBlock) {  // uniform
      const int seen = kb < pb ? pre_tail : sees(pos);
#pragma unroll
      for (int nb2 = 0; nb2 < 2; ++nb2)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * nb2 + 16 * (i / 8) + 8 * grp + i % 8 >= seen) s[nb2][i] = -__builtin_inff();
    }
#pragma unroll
    for (int nb2 = 0; nb2 < 2; ++nb2)
#pragma unroll
      for (int i = 0; i < 16; ++i) bmax = fmaxf(bmax, s[nb2][i]);
    bmax = fmaxf(bmax, xor_lanes_f32<32>(bmax)) * cq;
    if (__any(bmax - m_ref > kSlack)) {
      const float m_new = fmaxf(m_ref, fabsf(bmax) < kFar ? bmax - kDown : bmax);
      const float alpha = __builtin_amdgcn_exp2f(m_ref - m_new);
      m_ref = m_new;
      far = __any(m_ref > kNoMax && fabsf(m_ref) >= kFar);
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < DTL; ++d) o[d] *= alpha;
    }
    float c2 = cq;
    if (far) {  // uniform
      c2 = 1.0f;
#pragma unroll
      for (int nb2 = 0; nb2 < 2; ++nb2)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[nb2][i] *= cq;
    }
    // O^T over 4 steps of 16 keys, 8 of them this lane's; a step's weights are formed under the products of the one before
    float psum = 0.0f;
    v4i pf[2][NP];
    float v[8];
    auto read_scales = [&](int c) {
      if constexpr (!kScaled) {
        const float4 f0 = *reinterpret_cast<const float4*>(&svs[slot][16 * c + 8 * grp]);
        const float4 f1 = *reinterpret_cast<const float4*>(&svs[slot][16 * c + 8 * grp + 4]);
        v[0] = f0.x, v[1] = f0.y, v[2] = f0.z, v[3] = f0.w, v[4] = f1.x, v[5] = f1.y, v[6] = f1.z, v[7] = f1.w;
      }
    };
    auto weights = [&](int c, int j) {  // keys j and j + 1 of step c
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c / 2][8 * (c % 2) + j], c2, -m_ref));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c / 2][8 * (c % 2) + j + 1], c2, -m_ref));
      uint32_t part[NP];
      if constexpr (kScaled) {
        f16_parts<NP>(p0, p1, part);
        const f16x2_t one = {(_Float16)1.0f, (_Float16)1.0f};  // the sum of the weights as they are used
        psum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, part[0]), one, psum, false);
      } else {
        psum += p0;
        psum += p1;
        f16_parts<NP>(p0 * v[j], p1 * v[j + 1], part);
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) pf[c & 1][p][j / 2] = (int)part[p];
      asm volatile("" : "+v"(psum));  // here, under the products, not where the sum is used
    };
    v4i vf[kRingV];
    auto read_v = [&](int i) {
      vf[i % kRingV] = *reinterpret_cast<const v4i*>(
          &vs[32 * kKvBlock * (i % DTL) + va + 8 * ((2 * (i / DTL) + grp) ^ vx)]);
    };
    read_scales(0);
#pragma unroll
    for (int i = 0; i < kRingV; ++i) read_v(i);
#pragma unroll
    for (int j = 0; j < 8; j += 2) weights(0, j);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (c + 1 < 4) read_scales(c + 1);
#pragma unroll
      for (int d = 0; d < DTL; ++d) {
        const int i = c * DTL + d;
#pragma unroll
        for (int p = 0; p < NP; ++p)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, vf[i % kRingV]),
                                                        __builtin_bit_cast(f16x8_t, pf[c & 1][p]), o[d], 0, 0, 0);
        if (i + kRingV < 4 * DTL) read_v(i + kRingV);
        if (c + 1 < 4) {
#pragma unroll
          for (int j = 8 * d / DTL; j < 8 * (d + 1) / DTL; j += 2) weights(c + 1, j);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    l_run += psum;
  };

  if (kb0 < kb1) {
    stage_scales(0);
    sk = sk1;
    sv = sv1;
    stage_scales(1);
    fetch_scales(kb0 + 2 < kb1 ? kb0 + 2 : kb1 - 1);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      read_factors(i, 0);
#pragma unroll
      for (int x = 4 * i; x < 4 * i + 4; ++x) convert(x, 0);
      stage_codes(i, 0);
    }
    int slot = 0;
    for (int kb = kb0; kb < kb1; kb += 2) {
      __syncthreads();  // block kb and its scales are staged, and everyone is done with block kb - 1
      block(kb, 0, slot);
      slot = slot == 2 ? 0 : slot + 1;
      if (kb + 1 >= kb1) break;
      __syncthreads();
      block(kb + 1, 1, slot);
      slot = slot == 2 ? 0 : slot + 1;
    }
  }

  l_run += xor_lanes_f32<32>(l_run);
  // A lane holds O^T[32 d + 8 (i / 4) + 4 grp + i % 4] of its row.  Half a row at a time goes through LDS, so that it leaves
  // in one piece and not 16 bytes (of bf16 8) at a time.
  constexpr int NC = D / 8, RP = 64 / NC;  // pieces of four elements in half a row, rows that the wave stores at once
  // A part leaves as if its weights were at most one, so that a sum over values near the end of fp32 does not pass it (but
  // for far scores, where the shift need not be exact).
  constexpr float kOne = kSlack == 15.0f ? 0x1p-15f : 0x1p-1f;
  static_assert(kSlack == 15.0f || kSlack == 1.0f);
  const float down = far ? 1.0f : kOne;
  const float f = parts.o ? vref * (1.0f / kUp) * down : vref * (1.0f / kUp) / l_run;
  int64_t at = r < R ? qrow * a.ldo + (int64_t)h * D : -1;
  if (parts.o) {
    const int64_t row = (int64_t)(slot0 + split) * parts.rows + qrow * a.hq + h;
    at = valid ? row * D : -1;
    if (valid && grp == 0) parts.ml[row] = make_float2(far ? m_ref : m_ref + kSlack, l_run * down);
  }
  int64_t ats[32 / RP];  // of the rows that the lane stores a piece of
#pragma unroll
  for (int p = 0; p < 32 / RP; ++p) ats[p] = __shfl(at, p * RP + lane / NC);
  __syncthreads();  // no one reads the tiles any more
  float4* buf = reinterpret_cast<float4*>(tile) + w * 32 * NC;  // [row][piece ^ row]
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int d = 0; d < DTL / 2; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x16_t& x = o[half * (DTL / 2) + d];
        buf[col * NC + ((8 * d + i / 2 + grp) ^ (col % NC))] =
            valid ? make_float4(x[i] * f, x[i + 1] * f, x[i + 2] * f, x[i + 3] * f) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int p = 0; p < 32 / RP; ++p) {
      const int row = p * RP + lane / NC, piece = lane % NC;
      const float4 x = buf[row * NC + (piece ^ (row % NC))];
      const int64_t to = ats[p] + half * (D / 2) + 4 * piece;
      if (ats[p] < 0) continue;
      if (parts.o) {
        *reinterpret_cast<float4*>(parts.o + to) = x;
      } else {
        const float v[4] = {x.x, x.y, x.z, x.w};
        store4<DT>(a.out, to, v);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---- kernels ------------------------------------------------------------------------------------------

enum class Prefix { None, Columns, Rows };

// A decode step: the workgroups of the prefix, if there is one, then those of the sequences' own keys.
template <int DT, int D, Prefix P>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void kv_decode_kernel(KvAttn a, Parts parts,
                                                                                                     Plan plan) {
  using Own = DecodeShared<DT == WFB_F32 ? 3 : 2, D>;
  constexpr size_t kRowsBytes = P == Prefix::Rows ? sizeof(RowsShared<D>) : 0;
  __shared__ __attribute__((aligned(16))) char smem[kRowsBytes > sizeof(Own) ? kRowsBytes : sizeof(Own)];
  const int rows = a.b * (a.hq / a.hkv);
  int block = blockIdx.x;
  if constexpr (P != Prefix::None) {
    constexpr int kEach = P == Prefix::Rows ? 32 * kPrefixWaves : kColumns;
    const int nrb = (rows + kEach - 1) / kEach, mine = nrb * a.hkv * plan.pre;
    if (block < mine) {
      if constexpr (P == Prefix::Rows)
        rows_part<DT, D, kPrefixWaves, true>(a, parts, plan.own, plan.pre, block, *reinterpret_cast<RowsShared<D>*>(smem));
      else
        decode_part<DT, D, true>(a, parts, plan.own, plan.pre, block % a.hkv, block / a.hkv % nrb, block / a.hkv / nrb,
                                 *reinterpret_cast<Own*>(smem));
      return;
    }
    block -= mine;
  }
  decode_part<DT, D, false>(a, parts, 0, plan.own, block % a.hkv, block / a.hkv % a.b, block / a.hkv / a.b,
                            *reinterpret_cast<Own*>(smem));
}

template <int DT, int D, int W>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2))) void kv_rows_kernel(KvAttn a, Parts parts,
                                                                                                Plan plan) {
  __shared__ __attribute__((aligned(16))) RowsShared<D> sh;
  rows_part<DT, D, W, false>(a, parts, 0, plan.own, blockIdx.x, sh);
}

// ---- joining ----------------------------------------------------------------------------------------

// out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over the slots that were written, W waves per row: D / 4 lanes take
// four elements each, the groups of lanes the slots in turn.  Bound by latency (4 to 8 us for 1 to 30 MB).
template <int DT, int D, int W>
__global__ __launch_bounds__(kThreads) void kv_join_kernel(KvAttn a, Parts parts, Plan plan) {
  constexpr int L = D / 4, G = 64 * W / L;  // lanes of a group, groups of a row
  __shared__ float4 os[W > 1 ? G : 1][L];
  __shared__ float ls[W > 1 ? G : 1];
  const int t = threadIdx.x % (64 * W), lane = t & 63, j = t % L, g = t / L;
  const int64_t row = (int64_t)blockIdx.x * (4 / W) + __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * W));
  if (row >= parts.rows) return;  // (uniform over the waves of a row)
  const int h = (int)(row % a.hq), i = (int)(row / a.hq % a.t), b = (int)(row / a.hq / a.t);
  const int64_t out = ((int64_t)b * a.t + i) * a.ldo + (int64_t)h * D + 4 * j;
  int64_t first;
  int n;
  const bool fits = kv_span(a.span, b, first, n);
  if (!fits || i >= n) {
    const float x = fits ? 0.0f : __builtin_nanf(""), v[4] = {x, x, x, x};
    if (g == 0) store4<DT>(a.out, out, v);
    return;
  }
  int own = plan.own;
  if (plan.decode) {
    const int64_t nb = (first + kKvBlock - 1) / kKvBlock, per = split_blocks(nb, plan.own);
    own = nb == 0 ? 1 : (int)((nb + per - 1) / per);
  }
  int pre = plan.pre;
  if (plan.decode && !plan.pre_rows && pre > 0) {
    const int64_t nb = (a.npre + kKvBlock - 1) / kKvBlock, per = split_blocks(nb, pre);
    pre = (int)((nb + per - 1) / per);
  }
  const int total = own + pre;
  auto slot = [&](int s) { return (int64_t)(s < own ? s : plan.own + s - own) * parts.rows + row; };
  float m = kNoMax;
  for (int s = lane; s < total; s += 64) m = fmaxf(m, parts.ml[slot(s)].x);
  m = fmaxf(m, xor_lanes_f32<32>(m));
  m = fmaxf(m, xor_lanes_f32<16>(m));
  m = fmaxf(m, xor_lanes_f32<8>(m));
  m = fmaxf(m, xor_lanes_f32<4>(m));
  m = fmaxf(m, xor_lanes_f32<2>(m));
  m = fmaxf(m, xor_lanes_f32<1>(m));
  float l = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int s = g; s < total; s += G) {
    const int64_t at = slot(s);
    const float2 ml = parts.ml[at];
    const float4 x = *reinterpret_cast<const float4*>(parts.o + at * D + 4 * j);
    const float f = __builtin_amdgcn_exp2f(ml.x - m);
    l += ml.y * f;
    v[0] += x.x * f;
    v[1] += x.y * f;
    v[2] += x.z * f;
    v[3] += x.w * f;
  }
  if constexpr (W == 1) {
    // the groups of the wave: 2 of 32 lanes, or 4 of 16
    auto add = [&](float& x) {
      if constexpr (L == 16) x += xor_lanes_f32<16>(x);
      x += xor_lanes_f32<32>(x);
    };
    add(l);
#pragma unroll
    for (int e = 0; e < 4; ++e) add(v[e]);
  } else {
    os[g][j] = make_float4(v[0], v[1], v[2], v[3]);
    if (j == 0) ls[g] = l;
    __syncthreads();
    if (g > 0) return;
    l = 0.0f, v[0] = v[1] = v[2] = v[3] = 0.0f;
#pragma unroll
    for (int x = 0; x < G; ++x) {
      l += ls[x];
      v[0] += os[x][j].x;
      v[1] += os[x][j].y;
      v[2] += os[x][j].z;
      v[3] += os[x][j].w;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] /= l;
  if (g == 0) store4<DT>(a.out, out, v);
}

template <int DT, int D>
hipError_t launch_dd(const KvAttn& a, hipStream_t s) {
  // where starts are on the device, halfway between the first chunk of a cache and its last
  const int64_t cap = a.own.cap, keys = !a.span.start_dev ? a.span.start + a.t : a.t < cap ? (a.t + cap) / 2 : cap;
  const Plan p = make_plan(a.dt, a.b, a.t, a.hq, a.hkv, a.d, cap, keys, a.npre, a.span.len_dev != nullptr);
  const Parts parts = parts_of(a, p);
  const int g = a.hq / a.hkv;
  hipError_t e;
  if (p.decode) {
    const int rows = a.b * g, each = p.pre_rows ? 32 * kPrefixWaves : kColumns;
    const int64_t groups = (int64_t)a.hkv * a.b * p.own + (int64_t)(rows + each - 1) / each * a.hkv * p.pre;
    if (groups > INT32_MAX) return hipErrorInvalidValue;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(kThreads), 0, s, a, parts, p);
    };
    if (p.pre == 0) go(kv_decode_kernel<DT, D, Prefix::None>);
    else if (p.pre_rows) go(kv_decode_kernel<DT, D, Prefix::Rows>);
    else go(kv_decode_kernel<DT, D, Prefix::Columns>);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  } else {
    e = launch_kv_write_i8(a.dt, a.d, a.kn, a.ldk, a.vn, a.ldv, a.rc, a.rs, a.npre, a.own, a.span, a.b, a.hkv, s);
    if (e != hipSuccess) return e;
    const int each = 32 * p.waves;
    const int64_t groups = ((int64_t)a.t * g + each - 1) / each * a.hkv * a.b * p.own;
    if (groups > INT32_MAX) return hipErrorInvalidValue;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(64 * p.waves), 0, s, a, parts, p);
    };
    if (p.waves == kRowsWaves) go(kv_rows_kernel<DT, D, kRowsWaves>);
    else if constexpr (DT == WFB_BF16 || D == 64) go(kv_rows_kernel<DT, D, 4>);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (!has_parts(p)) return hipSuccess;
  // a row's slots by one wave, or by four where they are many: a whole call of 2 sequences of 8192 keys (32 splits of 64
  // rows) 16.0, 14.1 us; one of 4096 keys and 3 heads (16 splits) 9.5, 9.9; 4 of 8192 (16 splits of 128 rows) 20.5 both
  if (p.own + p.pre <= 16)
    hipLaunchKernelGGL((kv_join_kernel<DT, D, 1>), dim3((unsigned)((parts.rows + 3) / 4)), dim3(kThreads), 0, s, a, parts, p);
  else
    hipLaunchKernelGGL((kv_join_kernel<DT, D, 4>), dim3((unsigned)parts.rows), dim3(kThreads), 0, s, a, parts, p);
  return hipGetLastError();
}

}  // namespace

int64_t kv_attn_workspace_floats(int64_t b, int64_t t, int64_t hq, int64_t hkv, int64_t d, int64_t cap, int64_t npre) {
  // room for either type, and for one token per sequence with lengths, which takes the rows kernel
  int64_t most = 0;
  for (int dt : {WFB_F32, WFB_BF16})
    for (bool lengths : {false, true}) {
      const Plan p = make_plan(dt, b, t, hq, hkv, d, cap, cap, npre, lengths);
      if (has_parts(p)) most = most > p.own + p.pre ? most : p.own + p.pre;
    }
  return most * b * t * hq * (d + 2);
}

hipError_t launch_kv_attention(const KvAttn& a, hipStream_t s) {
  if (a.dt == WFB_F32) return a.d == 64 ? launch_dd<WFB_F32, 64>(a, s) : launch_dd<WFB_F32, 128>(a, s);
  return a.d == 64 ? launch_dd<WFB_BF16, 64>(a, s) : launch_dd<WFB_BF16, 128>(a, s);
}

}  // namespace wfb
