// Quantising write of new keys and values into the int8 cache, and the read back of a range of it.
#include "kv_i8.h"

namespace wfb {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// 4 x 4 bytes transposed: byte i of out[j] is byte j of in[i].
__device__ __forceinline__ void transpose4(const uint32_t (&in)[4], uint32_t (&out)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u);  // bytes 0.0 1.0 0.1 1.1
  const uint32_t b = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u);
  const uint32_t c = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);
  const uint32_t d = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
  out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
  out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
  out[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// Codes of 8 elements of a row held by the L = D / 8 lanes of a group, and the row's scale (the same in every lane).
template <int L>
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float& scale) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = umax(m, __float_as_uint(x[j]) & 0x7fffffffu);
  m = umax(m, (uint32_t)xor_lanes<1>((int)m));
  m = umax(m, (uint32_t)xor_lanes<2>((int)m));
  m = umax(m, (uint32_t)xor_lanes<4>((int)m));
  if constexpr (L == 16) m = umax(m, (uint32_t)xor_lanes<8>((int)m));
  float inv;
  kv_scale(m, scale, inv);
  uint32_t q[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j / 4] |= (uint32_t)(kv_code(x[j], inv) & 0xff) << 8 * (j % 4);
  return make_uint2(q[0], q[1]);
}

// One workgroup per (64-key block of the cache, kv head, sequence, keys or values): the new tokens that fall into the block.
// A row is read by D / 8 lanes, 8 elements each (the rotary partner D / 2 away sits in the lane half a group away); the
// value codes pass through LDS, row by row in and 4 x 4 bytes transposed out, 8 keys of 4 elements per thread.
// What bounds it, at 8 x 2048 tokens of 8 heads of 128: bf16, 67 MB in and 35 MB out in 29 us (3.5 TB/s; a copy of as many
// bytes takes 21), 27 without rotary tables; fp32, 134 MB in, 40 us (4.2 TB/s; a copy 33).  The 7 to 8 us over a copy are a
// workgroup's one chain of loads, maximum, codes and stores, in which only the CU's other workgroups keep memory busy.  With
// one workgroup for the keys and the values of a block, here and in the read back, the two calls took 58 us together, now 51.
template <int DT, int D>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(const void* __restrict__ kn, int64_t ldk,
                                                            const void* __restrict__ vn, int64_t ldv,
                                                            const float* __restrict__ rc, const float* __restrict__ rs,
                                                            int64_t turn, wfb_kv_i8 c, KvSpan sp, int hkv) {
  constexpr int HD = D / 2, L = D / 8, RPP = kThreads / L;  // lanes per row, rows per pass
  constexpr int NP = kKvBlock / RPP;                        // passes
  constexpr int kPitch = D + 8;                             // of an LDS row: the transposed reads spread over the banks
  __shared__ __attribute__((aligned(16))) uint8_t vt[kKvBlock * kPitch];
  const int t = threadIdx.x, l = t % L, h = blockIdx.y >> 1, b = blockIdx.z;
  const bool keys = (blockIdx.y & 1) == 0;
  int64_t first;
  int n;
  if (!kv_span(sp, b, first, n)) return;
  const int64_t k0 = (first / kKvBlock + blockIdx.x) * kKvBlock;
  // slots lo .. hi - 1 of the block
  const int lo = first > k0 ? (int)(first - k0) : 0;
  const int64_t left = first + n - k0;
  const int hi = left < kKvBlock ? (int)left : kKvBlock;
  if (lo >= hi) return;
  const int64_t slice = ((int64_t)b * hkv + h) * c.cap;
  const int64_t row0 = (int64_t)b * sp.t + (k0 - first);  // input row of slot 0
  auto at = [&](int p) {  // slot of pass p; one that is not written is read as the first that is
    const int slot = p * RPP + t / L;
    return slot >= lo && slot < hi ? slot : lo;
  };
  float x[NP][8];
#pragma unroll
  for (int p = 0; p < NP; ++p)
    if (p * RPP < hi && (p + 1) * RPP > lo)  // uniform
      load8<DT>(keys ? kn : vn, (row0 + at(p)) * (keys ? ldk : ldv) + (int64_t)h * D + 8 * l, x[p]);
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    if (p * RPP >= hi || (p + 1) * RPP <= lo) continue;
    const int slot = at(p);
    const int64_t pos = k0 + slot;
    if (keys && rc) {
      float cs[8], sn[8];
      load8<WFB_F32>(rc, (pos + turn) * HD + 8 * (l % (L / 2)), cs);
      load8<WFB_F32>(rs, (pos + turn) * HD + 8 * (l % (L / 2)), sn);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float other = xor_lanes_f32<L / 2>(x[p][j]);
        const float y = __fmul_rn(x[p][j], cs[j]), z = __fmul_rn(other, sn[j]);
        x[p][j] = l < L / 2 ? __fsub_rn(y, z) : __fadd_rn(y, z);
      }
    }
    float scale;
    const uint2 q = quantise8<L>(x[p], scale);
    if (slot == p * RPP + t / L) {
      if (keys) *reinterpret_cast<uint2*>(c.k + (slice + pos) * D + 8 * l) = q;
      else *reinterpret_cast<uint2*>(&vt[slot * kPitch + 8 * l]) = q;
      if (l == 0) (keys ? c.k_scale : c.v_scale)[slice + pos] = scale;
    }
  }
  if (keys) return;
  __syncthreads();
  int8_t* vb = c.v + (slice + k0) * D;
  for (int i = t; i < D / 4 * 8; i += kThreads) {
    const int s0 = 8 * (i % 8), d0 = 4 * (i / 8);
    if (s0 + 8 <= lo || s0 >= hi) continue;
    uint32_t q[2][4];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t in[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) in[r] = *reinterpret_cast<const uint32_t*>(&vt[(s0 + 4 * e + r) * kPitch + d0]);
      transpose4(in, q[e]);
    }
    const bool whole = s0 >= lo && s0 + 8 <= hi;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int8_t* dst = vb + (d0 + j) * kKvBlock + s0;
      if (whole) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(q[0][j], q[1][j]);
      } else {  // the block's other keys stay as they are
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (s0 + r >= lo && s0 + r < hi) dst[r] = (int8_t)(q[r / 4][j] >> 8 * (r % 4));
      }
    }
  }
}

// Four codes of a word as the values that they stand for: code = byte - 128 of the word with its sign bits flipped.
__device__ __forceinline__ void values4(uint32_t q, float scale, float (&v)[4]) {
  const uint32_t u = q ^ 0x80808080u;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = ((float)((u >> 8 * j) & 0xffu) - 128.0f) * scale;
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

// k / v [batch, kv_heads, count, D].  One workgroup per (64-key block, kv head, sequence, keys or values), the blocks counted
// from the one that holds the first position; positions outside the cache read as zeros.  A value block passes through
// LDS as it is stored and is read 4 keys x 4 elements at a time.
// What bounds it: memory.  8 x 2048 tokens of 8 heads of 128 that were just written: 35 MB in and 67 MB out as bf16 in 17 us
// (6.0 TB/s, above a copy's 4.9: part of the codes still lies in the last cache), 134 MB out as fp32 in 32 us (5.3 TB/s).
template <int DT, int D>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(wfb_kv_i8 c, const int64_t* __restrict__ start_dev, int64_t start,
                                                           int64_t count, int hkv, void* __restrict__ k,
                                                           void* __restrict__ v) {
  constexpr int kPitch = kKvBlock + 4;
  __shared__ __attribute__((aligned(16))) uint8_t vt[D * kPitch];
  __shared__ float vs[kKvBlock];
  const int t = threadIdx.x;
  const bool keys = (blockIdx.y & 1) == 0;
  const int64_t base = (int64_t)blockIdx.z * hkv + (blockIdx.y >> 1);
  int64_t first = start_dev ? start_dev[blockIdx.z] : start;
  first = first < -count ? -count : first > c.cap ? c.cap : first;  // (nothing inside on either side of these)
  constexpr int64_t kUp = int64_t(1) << 30;  // (first is above -2^24: rounded down to a block, not towards zero)
  const int64_t k0 = ((first + kUp) / kKvBlock + blockIdx.x) * kKvBlock - kUp;
  const int64_t from = first > k0 ? first - k0 : 0, left = first + count - k0;
  const int lo = from < kKvBlock ? (int)from : kKvBlock, hi = left < kKvBlock ? (int)left : kKvBlock;
  if (lo >= hi) return;
  const bool in = k0 >= 0 && k0 < c.cap;  // uniform (the capacity is a multiple of a block)
  const int64_t at = base * c.cap + (in ? k0 : 0), out0 = base * count + (k0 - first);  // output row of slot 0
  if (keys) {  // 16 elements per thread
    constexpr int L = D / 16;
#pragma unroll
    for (int p = 0; p < kKvBlock * L / kThreads; ++p) {
      const int i = t + p * kThreads, slot = i / L, d0 = 16 * (i % L);
      if (slot < lo || slot >= hi) continue;
      v4i q = {0, 0, 0, 0};
      float sc = 0.0f;
      if (in) {
        q = *reinterpret_cast<const v4i*>(c.k + (at + slot) * D + d0);
        sc = c.k_scale[at + slot];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x[4];
        values4((uint32_t)q[e], sc, x);
        store4<DT>(k, (out0 + slot) * D + d0 + 4 * e, x);
      }
    }
    return;
  }
  if (in) {
#pragma unroll
    for (int p = 0; p < D * 4 / kThreads; ++p) {
      const int i = t + p * kThreads;
      const v4i q = *reinterpret_cast<const v4i*>(c.v + at * D + 16 * i);
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<int*>(&vt[i / 4 * kPitch + 16 * (i % 4) + 4 * e]) = q[e];
    }
    if (t < kKvBlock) vs[t] = c.v_scale[at + t];
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < (D / 4) * (kKvBlock / 4) / kThreads; ++p) {
    const int i = t + p * kThreads, d0 = 4 * (i % (D / 4)), s0 = 4 * (i / (D / 4));
    if (s0 + 4 <= lo || s0 >= hi) continue;
    uint32_t q[4], r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = in ? *reinterpret_cast<const uint32_t*>(&vt[(d0 + j) * kPitch + s0]) : 0u;
    transpose4(q, r);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (s0 + e >= lo && s0 + e < hi) {
        float x[4];
        values4(r[e], in ? vs[s0 + e] : 0.0f, x);
        store4<DT>(v, (out0 + s0 + e) * D + d0, x);
      }
  }
}

}  // namespace

hipError_t launch_kv_write_i8(int dt, int d, const void* kn, int64_t ldk, const void* vn, int64_t ldv, const float* rc,
                              const float* rs, int64_t turn, const wfb_kv_i8& c, const KvSpan& sp, int b, int hkv,
                              hipStream_t s) {
  const dim3 grid((unsigned)((sp.t + kKvBlock - 2) / kKvBlock + 1), 2 * hkv, b);  // blocks that t positions can touch
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, kn, ldk, vn, ldv, rc, rs, turn, c, sp, hkv);
  };
  if (dt == WFB_F32) d == 64 ? go(kv_write_kernel<WFB_F32, 64>) : go(kv_write_kernel<WFB_F32, 128>);
  else d == 64 ? go(kv_write_kernel<WFB_BF16, 64>) : go(kv_write_kernel<WFB_BF16, 128>);
  return hipGetLastError();
}

hipError_t launch_kv_read_i8(int dt, int d, const wfb_kv_i8& c, const int64_t* start_dev, int64_t start, int b,
                             int64_t count, int hkv, void* k, void* v, hipStream_t s) {
  const dim3 grid((unsigned)((count + kKvBlock - 2) / kKvBlock + 1), 2 * hkv, b);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, c, start_dev, start, count, hkv, k, v);
  };
  if (dt == WFB_F32) d == 64 ? go(kv_read_kernel<WFB_F32, 64>) : go(kv_read_kernel<WFB_F32, 128>);
  else d == 64 ? go(kv_read_kernel<WFB_BF16, 64>) : go(kv_read_kernel<WFB_BF16, 128>);
  return hipGetLastError();
}

}  // namespace wfb
