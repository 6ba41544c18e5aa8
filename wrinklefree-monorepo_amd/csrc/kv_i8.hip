// Quantising write of new keys and values into the int8 cache, and the read back of a range of it.
#include "kv_i8.h"

namespace wfb {

namespace {

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  auto up = [&](uint32_t o) { v = o > v ? o : v; };
  up((uint32_t)xor_lanes<32>((int)v));
  up((uint32_t)xor_lanes<16>((int)v));
  up((uint32_t)xor_lanes<8>((int)v));
  up((uint32_t)xor_lanes<4>((int)v));
  up((uint32_t)xor_lanes<2>((int)v));
  up((uint32_t)xor_lanes<1>((int)v));
  return v;
}

// One wave per (token, kv head): its key and its value.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv_write_kernel(const void* __restrict__ kn, int64_t ldk,
                                                       const void* __restrict__ vn, int64_t ldv,
                                                       const float* __restrict__ rc, const float* __restrict__ rs,
                                                       int64_t turn, wfb_kv_i8 c, KvSpan sp, int hkv) {
  constexpr int HD = D / 2, E = D / 64;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t item = (int64_t)blockIdx.x * 4 + w;  // token * hkv + head
  const int b = blockIdx.y;
  int64_t first;
  int n;
  if (!kv_span(sp, b, first, n) || item >= (int64_t)n * hkv) return;
  const int64_t i = item / hkv, pos = first + i, row = (int64_t)b * sp.t + i;
  const int h = (int)(item % hkv);
  float x[2][E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    x[0][e] = load_elem<DT>(kn, row * ldk + (int64_t)h * D + lane + 64 * e);
    x[1][e] = load_elem<DT>(vn, row * ldv + (int64_t)h * D + lane + 64 * e);
  }
  if (rc) {
    const float* cp = rc + (pos + turn) * HD;
    const float* zp = rs + (pos + turn) * HD;
    if constexpr (E == 2) {
      const float a = x[0][0], y = x[0][1], cs = cp[lane], sn = zp[lane];
      x[0][0] = __fsub_rn(__fmul_rn(a, cs), __fmul_rn(y, sn));
      x[0][1] = __fadd_rn(__fmul_rn(y, cs), __fmul_rn(a, sn));
    } else {
      const float mine = x[0][0], other = xor_lanes_f32<32>(mine), cs = cp[lane & 31], sn = zp[lane & 31];
      const float p = __fmul_rn(mine, cs), r = __fmul_rn(other, sn);
      x[0][0] = lane < 32 ? __fsub_rn(p, r) : __fadd_rn(p, r);
    }
  }
  const int64_t base = (int64_t)b * hkv + h;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t u = __float_as_uint(x[kv][e]) & 0x7fffffffu;
      m = u > m ? u : m;
    }
    float scale, inv;
    kv_scale(wave_umax(m), scale, inv);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int8_t q = (int8_t)kv_code(x[kv][e], inv);
      const int j = lane + 64 * e;
      if (kv == 0) c.k[(base * c.cap + pos) * D + j] = q;
      else c.v[((base * c.cap + pos / kKvBlock * kKvBlock) * D) + (int64_t)j * kKvBlock + pos % kKvBlock] = q;
    }
    if (lane == 0) (kv == 0 ? c.k_scale : c.v_scale)[base * c.cap + pos] = scale;
  }
}

template <int DT>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float v) {
  if constexpr (DT == WFB_F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16_rne(v);
}

// k / v [batch, kv_heads, count, D]: positions outside the cache read as zeros
template <int DT, int D>
__global__ __launch_bounds__(256) void kv_read_kernel(wfb_kv_i8 c, const int64_t* __restrict__ start_dev, int64_t start,
                                                      int64_t count, int hkv, void* __restrict__ k,
                                                      void* __restrict__ v) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= count * D) return;
  const int64_t i = e / D, base = (int64_t)blockIdx.z * hkv + blockIdx.y;
  const int j = (int)(e % D);
  const int64_t first = start_dev ? start_dev[blockIdx.z] : start;
  const bool in = first < c.cap - i && first >= -i;
  const int64_t pos = in ? first + i : 0;
  const float kf = (float)c.k[(base * c.cap + pos) * D + j] * c.k_scale[base * c.cap + pos];
  const float vf = (float)c.v[((base * c.cap + pos / kKvBlock * kKvBlock) * D) + (int64_t)j * kKvBlock + pos % kKvBlock] *
                   c.v_scale[base * c.cap + pos];
  store_elem<DT>(k, base * count * D + e, in ? kf : 0.0f);
  store_elem<DT>(v, base * count * D + e, in ? vf : 0.0f);
}

}  // namespace

hipError_t launch_kv_write_i8(int dt, int d, const void* kn, int64_t ldk, const void* vn, int64_t ldv, const float* rc,
                              const float* rs, int64_t turn, const wfb_kv_i8& c, const KvSpan& sp, int b, int hkv,
                              hipStream_t s) {
  const dim3 grid((unsigned)((sp.t * hkv + 3) / 4), b);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, kn, ldk, vn, ldv, rc, rs, turn, c, sp, hkv); };
  if (dt == WFB_F32) d == 64 ? go(kv_write_kernel<WFB_F32, 64>) : go(kv_write_kernel<WFB_F32, 128>);
  else d == 64 ? go(kv_write_kernel<WFB_BF16, 64>) : go(kv_write_kernel<WFB_BF16, 128>);
  return hipGetLastError();
}

hipError_t launch_kv_read_i8(int dt, int d, const wfb_kv_i8& c, const int64_t* start_dev, int64_t start, int b,
                             int64_t count, int hkv, void* k, void* v, hipStream_t s) {
  const dim3 grid((unsigned)((count * d + 255) / 256), hkv, b);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, c, start_dev, start, count, hkv, k, v); };
  if (dt == WFB_F32) d == 64 ? go(kv_read_kernel<WFB_F32, 64>) : go(kv_read_kernel<WFB_F32, 128>);
  else d == 64 ? go(kv_read_kernel<WFB_BF16, 64>) : go(kv_read_kernel<WFB_BF16, 128>);
  return hipGetLastError();
}

}  // namespace wfb
