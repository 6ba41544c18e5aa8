// RMSNorm of every query and key head with the rotary embedding of its position, and the backward pass, each in one pass.
//
//   n = x r,  r = (mean(x^2) + eps)^(-1/2),  y = n w          (no weight: y = x)
//   out = y with pair (a, b) of its first R elements turned by the angle of its position: (a c - b s, b c + a s)
//   g' = the gradient with its pairs turned back,  grad_w = sum over rows of g' n
//   grad_x = r (g' w - n mean(g' w n))                          (no weight: grad_x = g')
// Statistics, rotation and sums are fp32; each result is rounded once to its type.
//
// The rotation itself is the reference's training attention's (WF/models/attention.py:14-64, adjacent elements paired)
// and the stage-1 model's (halves paired); the norm of each head has no counterpart there.
#include "train_ops.h"

namespace wfb {

namespace {

// Elements travel in chunks of V (one load each, 16 bytes where the sizes allow it).  Item j of a row is two chunks
// that hold V whole pairs, chunk j of each half of the rotated part or two neighbours (interleaved layout); behind the
// rotated part, two neighbours that pass.  A row takes L lanes (a power of two), IT items each.  A group of lanes walks
// kHeads heads of one token, which share the angles.
constexpr int kThreads = 256;
constexpr int kHeads = 4;

template <int DT, int V>
__device__ __forceinline__ void load_chunk(const void* p, int64_t i, float* v) {
  if constexpr (DT == WFB_F32) {
    const float* q = reinterpret_cast<const float*>(p) + i;
    if constexpr (V % 4 == 0) {
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        const float4 x = *reinterpret_cast<const float4*>(q + e);
        v[e] = x.x, v[e + 1] = x.y, v[e + 2] = x.z, v[e + 3] = x.w;
      }
    } else if constexpr (V == 2) {
      const float2 x = *reinterpret_cast<const float2*>(q);
      v[0] = x.x, v[1] = x.y;
    } else {
      v[0] = q[0];
    }
  } else if constexpr (V == 1) {
    v[0] = load_elem<DT>(p, i);
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p) + i;
    uint32_t w[V / 2];
    if constexpr (V == 8) {
      const uint4 x = *reinterpret_cast<const uint4*>(q);
      w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
    } else if constexpr (V == 4) {
      const uint2 x = *reinterpret_cast<const uint2*>(q);
      w[0] = x.x, w[1] = x.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(q);
    }
#pragma unroll
    for (int e = 0; e < V / 2; ++e) {
      if constexpr (DT == WFB_BF16) {
        v[2 * e] = __uint_as_float(w[e] << 16);
        v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
      } else {
        v[2 * e] = f16_bits_to_f32((uint16_t)(w[e] & 0xffffu));
        v[2 * e + 1] = f16_bits_to_f32((uint16_t)(w[e] >> 16));
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ uint32_t half_bits(float v) {
  if constexpr (DT == WFB_BF16) return f32_to_bf16_rne(v);
  else return __builtin_bit_cast(uint16_t, (_Float16)v);
}

template <int DT, int V>
__device__ __forceinline__ void store_chunk(void* p, int64_t i, const float* v) {
  if constexpr (DT == WFB_F32) {
    float* q = reinterpret_cast<float*>(p) + i;
    if constexpr (V % 4 == 0) {
#pragma unroll
      for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(q + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else if constexpr (V == 2) {
      *reinterpret_cast<float2*>(q) = make_float2(v[0], v[1]);
    } else {
      q[0] = v[0];
    }
  } else if constexpr (V == 1) {
    reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)half_bits<DT>(v[0]);
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(p) + i;
    uint32_t w[V / 2];
#pragma unroll
    for (int e = 0; e < V / 2; ++e) w[e] = half_bits<DT>(v[2 * e]) | half_bits<DT>(v[2 * e + 1]) << 16;
    if constexpr (V == 8) *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (V == 4) *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(q) = w[0];
  }
}

__device__ __forceinline__ float load_weight(const void* w, int wdt, int i) {
  if (wdt == WFB_F32) return load_elem<WFB_F32>(w, i);
  return wdt == WFB_BF16 ? load_elem<WFB_BF16>(w, i) : load_elem<WFB_F16>(w, i);
}

// Where item j lies: its two chunks' first elements and its first pair, -1 behind the rotated part.
template <int V>
__device__ __forceinline__ void item_place(const QkRope& p, int j, int& ea, int& eb, int& pair) {
  const int turned = p.rotary / (2 * V);
  if (j >= turned) {
    ea = p.rotary + 2 * V * (j - turned);
    eb = ea + V;
    pair = -1;
  } else {
    pair = j * V;
    ea = p.interleaved ? 2 * V * j : V * j;
    eb = p.interleaved ? ea + V : ea + p.rotary / 2;
  }
}

// The 2V elements x (chunk a, then chunk b) turned by the angles c, s; back: by their negatives.
template <int V>
__device__ __forceinline__ void turn(float (&x)[2 * V], const float (&c)[V], const float (&s)[V], bool interleaved,
                                     bool back) {
  if (interleaved) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float sn = back ? -s[e] : s[e], a = x[2 * e], b = x[2 * e + 1];
      x[2 * e] = a * c[e] - b * sn;
      x[2 * e + 1] = b * c[e] + a * sn;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float sn = back ? -s[e] : s[e], a = x[e], b = x[V + e];
      x[e] = a * c[e] - b * sn;
      x[V + e] = b * c[e] + a * sn;
    }
  }
}

// What a group of lanes works on: kHeads heads from `head` on of one side at token (b, t).
struct Task {
  int side, head, count;
  int64_t b, t;
};

// (fewer than 2^31 tasks, host-checked: 32-bit divisions)
__device__ __forceinline__ Task task_of(const QkRope& p, uint32_t i) {
  const int cq = (p.side[0].heads + kHeads - 1) / kHeads, ck = (p.side[1].heads + kHeads - 1) / kHeads;
  const uint32_t token = i / (uint32_t)(cq + ck), bi = token / (uint32_t)p.t;
  const int c = (int)(i - token * (uint32_t)(cq + ck));
  Task k;
  k.side = c >= cq;
  k.head = (k.side ? c - cq : c) * kHeads;
  k.count = min(kHeads, (k.side ? p.side[1].heads : p.side[0].heads) - k.head);
  k.b = bi;
  k.t = token - bi * (uint32_t)p.t;
  return k;
}

__device__ __forceinline__ int64_t position_of(const QkRope& p, const Task& k) {
  if (!p.pos) return p.start + k.t;
  const int64_t i = k.b * p.pb + k.t * p.pt;
  return p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[i] : reinterpret_cast<const int32_t*>(p.pos)[i];
}

template <int V>
__device__ __forceinline__ void load_angles(const QkRope& p, int64_t at, int pair, float (&c)[V], float (&s)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) c[e] = 1.0f, s[e] = 0.0f;
  if (pair < 0) return;
  if (at < 0 || at >= p.rope_len) {  // no such position: the row becomes NaN, and nothing is read
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = s[e] = __builtin_nanf("");
    return;
  }
  load_chunk<WFB_F32, V>(p.cos, at * (p.rotary / 2) + pair, c);
  load_chunk<WFB_F32, V>(p.sin, at * (p.rotary / 2) + pair, s);
}

template <int DT, int V, int L, int IT>
__global__ __launch_bounds__(kThreads) void qk_rope_kernel(QkRope p, uint32_t tasks) {
  const int lane = threadIdx.x % L;
  const uint32_t i = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const bool live = i < tasks;
  const Task k = task_of(p, live ? i : 0);
  const HeadRows sd = k.side ? p.side[1] : p.side[0];
  const int D = p.head_dim, items = D / (2 * V);
  const int64_t at = position_of(p, k);
  const bool lost = p.rotary > 0 && (at < 0 || at >= p.rope_len);
  float x[IT][kHeads][2 * V];
  int ea[IT], eb[IT], pair[IT];
  bool on[IT];
  const int64_t row = k.b * sd.xb + k.t * sd.xt + k.head * sd.xh;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int j = lane + L * it;
    on[it] = live && j < items;
    item_place<V>(p, on[it] ? j : 0, ea[it], eb[it], pair[it]);
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) x[it][h][e] = 0.0f;
      if (on[it] && h < k.count) {
        load_chunk<DT, V>(sd.x, row + h * sd.xh + ea[it], &x[it][h][0]);
        load_chunk<DT, V>(sd.x, row + h * sd.xh + eb[it], &x[it][h][V]);
      }
    }
  }
  float w[IT][2 * V], c[IT][V], s[IT][V];
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    load_angles<V>(p, at, on[it] ? pair[it] : -1, c[it], s[it]);
#pragma unroll
    for (int e = 0; e < 2 * V; ++e) w[it][e] = 1.0f;
    if (sd.w && on[it]) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        w[it][e] = load_weight(sd.w, sd.wdt, ea[it] + e);
        w[it][V + e] = load_weight(sd.w, sd.wdt, eb[it] + e);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    float r = 1.0f;
    if (sd.w) {  // (the lanes of a row agree)
      float ss = 0.0f;
#pragma unroll
      for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) ss += x[it][h][e] * x[it][h][e];
#pragma unroll
      for (int o = 1; o < L; o <<= 1) ss += __shfl_xor(ss, o, 64);
      r = 1.0f / sqrtf(ss / (float)D + p.eps);
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      if (!on[it] || h >= k.count) continue;
      float y[2 * V];
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) y[e] = x[it][h][e] * r * w[it][e];
      if (pair[it] >= 0) turn<V>(y, c[it], s[it], p.interleaved, false);
      if (lost) {
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) y[e] = __builtin_nanf("");
      }
      const int64_t o = ((k.b * p.t + k.t) * sd.heads + k.head + h) * D;
      store_chunk<DT, V>(sd.out, o + ea[it], &y[0]);
      store_chunk<DT, V>(sd.out, o + eb[it], &y[V]);
    }
  }
}

template <int DT, int V, int L, int IT>
__global__ __launch_bounds__(kThreads) void qk_rope_grad_kernel(QkRope p, uint32_t tasks, float* __restrict__ part) {
  __shared__ float red[kThreads / L][2 * V * IT * L];
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  const int D = p.head_dim, items = D / (2 * V);
  float acc[2][IT][2 * V];
#pragma unroll
  for (int sdx = 0; sdx < 2; ++sdx)
#pragma unroll
    for (int it = 0; it < IT; ++it)
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) acc[sdx][it][e] = 0.0f;
  int ea[IT], eb[IT], pair[IT];
#pragma unroll
  for (int it = 0; it < IT; ++it) item_place<V>(p, min(lane + L * it, items - 1), ea[it], eb[it], pair[it]);

  // every group of the workgroup takes the same number of turns, so that the lanes of a wave stay together
  constexpr int G = kThreads / L;
  for (uint32_t i0 = blockIdx.x * G; i0 < tasks; i0 += gridDim.x * G) {
    const bool live = i0 + grp < tasks;
    const Task k = task_of(p, live ? i0 + grp : 0);
    const HeadRows sd = k.side ? p.side[1] : p.side[0];
    const int64_t at = position_of(p, k);
    const bool lost = p.rotary > 0 && (at < 0 || at >= p.rope_len);
    const int64_t row = k.b * sd.xb + k.t * sd.xt + k.head * sd.xh, grow = k.b * sd.gb + k.t * sd.gt + k.head * sd.gh;
    float c[IT][V], s[IT][V], w[IT][2 * V];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const bool on = live && lane + L * it < items;
      load_angles<V>(p, at, on ? pair[it] : -1, c[it], s[it]);
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) w[it][e] = 1.0f;
      if (sd.w && on) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          w[it][e] = load_weight(sd.w, sd.wdt, ea[it] + e);
          w[it][V + e] = load_weight(sd.w, sd.wdt, eb[it] + e);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      float x[IT][2 * V], g[IT][2 * V];
      float ss = 0.0f, sg = 0.0f;
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const bool on = live && lane + L * it < items && h < k.count;
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) x[it][e] = g[it][e] = 0.0f;
        if (on) {
          load_chunk<DT, V>(sd.g, grow + h * sd.gh + ea[it], &g[it][0]);
          load_chunk<DT, V>(sd.g, grow + h * sd.gh + eb[it], &g[it][V]);
          if (sd.w) {
            load_chunk<DT, V>(sd.x, row + h * sd.xh + ea[it], &x[it][0]);
            load_chunk<DT, V>(sd.x, row + h * sd.xh + eb[it], &x[it][V]);
          }
          if (pair[it] >= 0) turn<V>(g[it], c[it], s[it], p.interleaved, true);
          if (lost) {
#pragma unroll
            for (int e = 0; e < 2 * V; ++e) g[it][e] = __builtin_nanf("");
          }
        }
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          ss += x[it][e] * x[it][e];
          sg += g[it][e] * w[it][e] * x[it][e];
        }
      }
      float r = 1.0f, m = 0.0f;
      if (sd.w) {
#pragma unroll
        for (int o = 1; o < L; o <<= 1) {
          ss += __shfl_xor(ss, o, 64);
          sg += __shfl_xor(sg, o, 64);
        }
        r = 1.0f / sqrtf(ss / (float)D + p.eps);
        m = r * (sg / (float)D);
      }
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const bool on = live && lane + L * it < items && h < k.count;
        float y[2 * V];
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          const float n = x[it][e] * r, d = g[it][e] * n;
          y[e] = sd.w ? r * (g[it][e] * w[it][e] - n * m) : g[it][e];
          acc[0][it][e] += k.side ? 0.0f : d;
          acc[1][it][e] += k.side ? d : 0.0f;
        }
        if (on && sd.out) {
          const int64_t o = ((k.b * p.t + k.t) * sd.heads + k.head + h) * D;
          store_chunk<DT, V>(sd.out, o + ea[it], &y[0]);
          store_chunk<DT, V>(sd.out, o + eb[it], &y[V]);
        }
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int sdx = 0; sdx < 2; ++sdx) {
    if (sdx) __syncthreads();
#pragma unroll
    for (int it = 0; it < IT; ++it)
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) red[grp][(it * 2 * V + e) * L + lane] = acc[sdx][it][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * V * IT * L; i += kThreads) {
      float v = 0.0f;
      for (int q = 0; q < G; ++q) v += red[q][i];
      const int ln = i % L, e = i / L % (2 * V), it = i / L / (2 * V), j = ln + L * it;
      if (j >= items) continue;
      int a, b, pr;
      item_place<V>(p, j, a, b, pr);
      part[((int64_t)blockIdx.x * 2 + sdx) * D + (e < V ? a + e : b + e - V)] = v;
    }
  }
}

constexpr int kGradGroups = 512;

// The widest chunk that the sizes, strides and addresses allow: whole pairs on either side of the rotated part's end,
// chunks that start at multiples of their length in every row, and in the tables' rows.
int chunk_of(const QkRope& p, int dtype, bool grad) {
  const int esz = dtype == WFB_F32 ? 4 : 2;
  auto fits = [&](int v) {
    if (p.rotary % (2 * v) || (p.head_dim - p.rotary) % (2 * v)) return false;
    auto whole = [&](const void* q, int64_t a, int64_t b, int64_t c) {
      return (uintptr_t)q % (v * esz) == 0 && a % v == 0 && b % v == 0 && c % v == 0;
    };
    for (const HeadRows& s : p.side) {
      if (!whole(s.x, s.xb, s.xt, s.xh) || !whole(s.out, 0, 0, 0)) return false;
      if (grad && !whole(s.g, s.gb, s.gt, s.gh)) return false;
    }
    const int tv = v >= 4 ? 16 : 4 * v;
    return p.rotary == 0 || ((uintptr_t)p.cos % tv == 0 && (uintptr_t)p.sin % tv == 0);
  };
  for (int v = dtype == WFB_F32 ? 4 : 8; v > 1; v /= 2)
    if (fits(v)) return v;
  return 1;
}

template <int DT, int V, int L, int IT>
hipError_t launch(const QkRope& p, bool grad, float* part, int groups, hipStream_t s) {
  const int64_t tasks = qk_tasks(p);
  if (!grad) {
    const int64_t grid = (tasks + kThreads / L - 1) / (kThreads / L);
    hipLaunchKernelGGL((qk_rope_kernel<DT, V, L, IT>), dim3((unsigned)grid), dim3(kThreads), 0, s, p, (uint32_t)tasks);
  } else {
    hipLaunchKernelGGL((qk_rope_grad_kernel<DT, V, L, IT>), dim3((unsigned)groups), dim3(kThreads), 0, s, p, (uint32_t)tasks, part);
  }
  return hipGetLastError();
}

// Lanes of a row: the least power of two that holds its items, 8 at least.
template <int DT>
hipError_t dispatch(const QkRope& p, int v, bool grad, float* part, int groups, hipStream_t s) {
  const int items = p.head_dim / (2 * v);
  if constexpr (DT != WFB_F32) {
    if (v == 8) {
      if (items <= 8) return launch<DT, 8, 8, 1>(p, grad, part, groups, s);
      return launch<DT, 8, 16, 1>(p, grad, part, groups, s);
    }
  }
  if (v == 4) {
    if (items <= 8) return launch<DT, 4, 8, 1>(p, grad, part, groups, s);
    if (items <= 16) return launch<DT, 4, 16, 1>(p, grad, part, groups, s);
    return launch<DT, 4, 32, 1>(p, grad, part, groups, s);
  }
  if (v == 2) {
    if (items <= 16) return launch<DT, 2, 16, 1>(p, grad, part, groups, s);
    if (items <= 32) return launch<DT, 2, 32, 1>(p, grad, part, groups, s);
    return launch<DT, 2, 64, 1>(p, grad, part, groups, s);
  }
  return launch<DT, 1, 64, 2>(p, grad, part, groups, s);
}

hipError_t dispatch_type(const QkRope& p, int dtype, bool grad, float* part, int groups, hipStream_t s) {
  const int v = chunk_of(p, dtype, grad);
  if (dtype == WFB_F32) return dispatch<WFB_F32>(p, v, grad, part, groups, s);
  if (dtype == WFB_BF16) return dispatch<WFB_BF16>(p, v, grad, part, groups, s);
  return dispatch<WFB_F16>(p, v, grad, part, groups, s);
}

// The weights' gradients: the sums over the rows of part[rows][2][D], in a fixed order.  16 x 16 threads: 16 columns.
__global__ __launch_bounds__(256) void qk_weight_sum_kernel(const float* __restrict__ part, int rows, int D,
                                                            void* __restrict__ o0, int dt0, void* __restrict__ o1,
                                                            int dt1) {
  __shared__ float red[16][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, col = blockIdx.x * 16 + c, cc = min(col, 2 * D - 1);
  float acc = 0.0f;
  for (int i = r; i < rows; i += 16 * 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = part[(int64_t)min(i + 16 * u, rows - 1) * 2 * D + cc];
#pragma unroll
    for (int u = 0; u < 8; ++u) acc += i + 16 * u < rows ? v[u] : 0.0f;
  }
  red[r][c] = acc;
  __syncthreads();
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) {
    if (r < o) red[r][c] += red[r + o][c];
    __syncthreads();
  }
  if (r != 0 || col >= 2 * D) return;
  void* out = col < D ? o0 : o1;
  const int dt = col < D ? dt0 : dt1, i = col < D ? col : col - D;
  if (!out) return;
  if (dt == WFB_F32) reinterpret_cast<float*>(out)[i] = red[0][c];
  else if (dt == WFB_BF16) reinterpret_cast<uint16_t*>(out)[i] = f32_to_bf16_rne(red[0][c]);
  else reinterpret_cast<uint16_t*>(out)[i] = __builtin_bit_cast(uint16_t, (_Float16)red[0][c]);
}

}  // namespace

int64_t qk_tasks(const QkRope& p) {
  return p.batch * p.t * ((p.side[0].heads + kHeads - 1) / kHeads + (p.side[1].heads + kHeads - 1) / kHeads);
}

int qk_grad_parts(const QkRope& p) {
  // at least four groups of lanes a workgroup: more workgroups than that have nothing to do
  const int64_t most = (qk_tasks(p) + 3) / 4;
  return (int)(most < kGradGroups ? most : kGradGroups);
}

hipError_t launch_qk_rope(const QkRope& p, int dtype, hipStream_t s) { return dispatch_type(p, dtype, false, nullptr, 0, s); }

hipError_t launch_qk_rope_grad(const QkRope& p, int dtype, void* gw0, int gdt0, void* gw1, int gdt1, float* work,
                               hipStream_t s) {
  const int groups = qk_grad_parts(p), D = p.head_dim;
  const bool sums = gw0 || gw1;
  // (no rows: the weights' gradients are sums of nothing)
  const hipError_t e = groups ? dispatch_type(p, dtype, true, sums ? work : nullptr, groups, s) : hipSuccess;
  if (e != hipSuccess || !sums) return e;
  hipLaunchKernelGGL(qk_weight_sum_kernel, dim3((2 * D + 15) / 16), dim3(256), 0, s, work, groups, D, gw0, gdt0, gw1,
                     gdt1);
  return hipGetLastError();
}

}  // namespace wfb
