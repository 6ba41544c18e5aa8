// GQA attention over the int8 key/value cache (kv_i8.h): softmax(rope(q) . k * scale) v over the keys of a shared prefix
// and a sequence's own keys up to the query's position.
#include "kv_i8.h"

namespace wfb {

namespace {

template <int DT>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float v) {
  if constexpr (DT == WFB_F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16_rne(v);
}

// One workgroup per (query head, token): scores of 256 keys at a time, a running softmax, the weighted sum of values
// with the threads over (element, key residue).
template <int DT, int D>
__global__ __launch_bounds__(256) void kv_attention_kernel(KvAttn a) {
  constexpr int HD = D / 2, NG = 256 / D;
  __shared__ float qs[D], ps[256], red[4], acc_s[NG][D];
  const int h = blockIdx.x, i = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
  const int64_t row = (int64_t)b * a.t + i;
  int64_t first;
  int n;
  const bool fits = kv_span(a.span, b, first, n);
  if (!fits || i >= n) {
    if (t < D) store_elem<DT>(a.out, row * a.ldo + (int64_t)h * D + t, fits ? 0.0f : __builtin_nanf(""));
    return;
  }
  const int64_t pos = first + i;
  const int kvh = h / (a.hq / a.hkv);
  if (t < HD) {
    float x1 = load_elem<DT>(a.q, row * a.ldq + (int64_t)h * D + t);
    float x2 = load_elem<DT>(a.q, row * a.ldq + (int64_t)h * D + t + HD);
    if (a.rc) {
      const float cs = a.rc[(pos + a.npre) * HD + t], sn = a.rs[(pos + a.npre) * HD + t];
      const float y1 = __fsub_rn(__fmul_rn(x1, cs), __fmul_rn(x2, sn));
      x2 = __fadd_rn(__fmul_rn(x2, cs), __fmul_rn(x1, sn));
      x1 = y1;
    }
    qs[t] = x1 * a.scale;
    qs[t + HD] = x2 * a.scale;
  }
  __syncthreads();
  float m = -1e30f, l = 0.0f, acc = 0.0f;
  for (int part = 0; part < 2; ++part) {
    const wfb_kv_i8& c = part ? a.own : a.pre;
    const int64_t keys = part ? pos + 1 : a.npre, base = part ? (int64_t)b * a.hkv + kvh : kvh;
    for (int64_t k0 = 0; k0 < keys; k0 += 256) {
      const int64_t key = k0 + t;
      float s = -__builtin_inff();
      if (key < keys) {
        const int8_t* kr = c.k + (base * c.cap + key) * D;
        float dot = 0.0f;
        for (int e = 0; e < D; ++e) dot += qs[e] * (float)kr[e];
        s = dot * c.k_scale[base * c.cap + key];
      }
      float mx = s;
      mx = fmaxf(mx, xor_lanes_f32<32>(mx));
      mx = fmaxf(mx, xor_lanes_f32<16>(mx));
      mx = fmaxf(mx, xor_lanes_f32<8>(mx));
      mx = fmaxf(mx, xor_lanes_f32<4>(mx));
      mx = fmaxf(mx, xor_lanes_f32<2>(mx));
      mx = fmaxf(mx, xor_lanes_f32<1>(mx));
      __syncthreads();
      if (t % 64 == 0) red[t / 64] = mx;
      __syncthreads();
      const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
      const float al = __expf(m - mn), p = __expf(s - mn);
      m = mn;
      l = l * al + p;  // this thread's keys
      ps[t] = key < keys ? p * c.v_scale[base * c.cap + key] : 0.0f;
      __syncthreads();
      acc *= al;
      const int8_t* vb = c.v + (base * c.cap + k0) * D + (t % D) * kKvBlock;
      for (int j = t / D; j < 256 && k0 + j < keys; j += NG)
        acc += ps[j] * (float)vb[(j / kKvBlock) * kKvBlock * D + j % kKvBlock];
    }
  }
  acc_s[t / D][t % D] = acc;
  l = group_sum_f32<64>(l);
  __syncthreads();
  if (t % 64 == 0) red[t / 64] = l;
  __syncthreads();
  if (t < D) {
    float o = 0.0f;
    for (int g = 0; g < NG; ++g) o += acc_s[g][t];
    store_elem<DT>(a.out, row * a.ldo + (int64_t)h * D + t, o / ((red[0] + red[1]) + (red[2] + red[3])));
  }
}

}  // namespace

int64_t kv_attn_workspace_floats(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

hipError_t launch_kv_attention(const KvAttn& a, hipStream_t s) {
  hipError_t e = launch_kv_write_i8(a.dt, a.d, a.kn, a.ldk, a.vn, a.ldv, a.rc, a.rs, a.npre, a.own, a.span, a.b, a.hkv, s);
  if (e != hipSuccess) return e;
  const dim3 grid(a.hq, a.t, a.b);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, a); };
  if (a.dt == WFB_F32) a.d == 64 ? go(kv_attention_kernel<WFB_F32, 64>) : go(kv_attention_kernel<WFB_F32, 128>);
  else a.d == 64 ? go(kv_attention_kernel<WFB_BF16, 64>) : go(kv_attention_kernel<WFB_BF16, 128>);
  return hipGetLastError();
}

}  // namespace wfb
