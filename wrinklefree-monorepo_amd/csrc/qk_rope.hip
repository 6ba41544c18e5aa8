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
// kHeads heads of one token, which share the angles; all their loads are requested before the first is used, and stay as
// they were loaded until they are.
constexpr int kThreads = 256;
constexpr int kHeads = 4;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// V elements of type DT as the words they are loaded in (V = 1 of 16 bits: one half of a word).
template <int DT, int V>
struct Chunk {
  static constexpr int N = DT == WFB_F32 ? V : (V + 1) / 2;
  uint32_t w[N];

  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if constexpr (DT != WFB_F32 && V == 1) {
      w[0] = reinterpret_cast<const uint16_t*>(p)[i];
    } else {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(reinterpret_cast<const char*>(p) + i * (DT == WFB_F32 ? 4 : 2));
      if constexpr (N % 4 == 0) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(q + e);
          w[e] = x.x, w[e + 1] = x.y, w[e + 2] = x.z, w[e + 3] = x.w;
        }
      } else if constexpr (N == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(q);
        w[0] = x.x, w[1] = x.y;
      } else {
        w[0] = q[0];
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = 0;
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (DT == WFB_F32) return __uint_as_float(w[e]);
    else if constexpr (DT == WFB_BF16) return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    else return f16_bits_to_f32((uint16_t)(w[e / 2] >> (16 * (e & 1))));
  }
};

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == WFB_BF16) return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
  else return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
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
    reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)pack2<DT>(v[0], 0.0f);
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(p) + i;
    uint32_t w[V / 2];
#pragma unroll
    for (int e = 0; e < V / 2; ++e) w[e] = pack2<DT>(v[2 * e], v[2 * e + 1]);
    if constexpr (V == 8) *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (V == 4) *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(q) = w[0];
  }
}

template <int WDT, int V>
__device__ __forceinline__ void load_weight(const void* w, int ea, int eb, float (&v)[2 * V]) {
  Chunk<WDT, V> a, b;
  a.load(w, ea);
  b.load(w, eb);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = a.get(e), v[V + e] = b.get(e);
}

// The norm's weight for an item, ones without a norm.
template <int V>
__device__ __forceinline__ void item_weight(const HeadRows& s, bool on, int ea, int eb, float (&v)[2 * V]) {
#pragma unroll
  for (int e = 0; e < 2 * V; ++e) v[e] = 1.0f;
  if (!s.w || !on) return;
  if (s.wdt == WFB_F32) load_weight<WFB_F32, V>(s.w, ea, eb, v);
  else if (s.wdt == WFB_BF16) load_weight<WFB_BF16, V>(s.w, ea, eb, v);
  else load_weight<WFB_F16, V>(s.w, ea, eb, v);
}

// Sum over a row's L lanes, in every one of them.  (Lanes of other rows may be elsewhere: their side has no norm.)
template <int L>
__device__ __forceinline__ float row_sum(float v) {
  if constexpr (L <= 16) {
    return group_sum_f32<L>(v);
  } else {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
  }
}

// v^(-1/2), root and quotient each correctly rounded, subnormal v too.  (The one-instruction form is off by an ulp and takes
// subnormal numbers for 0; either way the passes wait for memory: TIMES)
__device__ __forceinline__ float inverse_root(float v) { return __fdiv_rn(1.0f, sqrtf(v)); }

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

// The 2V elements x (chunk a, then chunk b) turned by the angles c, s (of the opposite sign to turn back).
template <int V>
__device__ __forceinline__ void turn(float (&x)[2 * V], const float (&c)[V], const float (&s)[V], bool interleaved) {
  if (interleaved) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = x[2 * e], b = x[2 * e + 1];
      x[2 * e] = __builtin_fmaf(a, c[e], -(b * s[e]));
      x[2 * e + 1] = __builtin_fmaf(b, c[e], a * s[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = x[e], b = x[V + e];
      x[e] = __builtin_fmaf(a, c[e], -(b * s[e]));
      x[V + e] = __builtin_fmaf(b, c[e], a * s[e]);
    }
  }
}

// What a group of lanes works on: kHeads heads from `head` on of one side at token (b, t).
struct Task {
  int head, count;
  int64_t b, t;
};

// Task i of the tokens' groups of heads, `chunks` of them a token.  (fewer than 2^31 tasks, host-checked: 32-bit divisions)
__device__ __forceinline__ Task task_of(uint32_t i, uint32_t chunks, int heads, uint32_t tokens) {
  const uint32_t token = i / chunks, bi = token / tokens;
  Task k;
  k.head = (int)(i - token * chunks) * kHeads;
  k.count = min(kHeads, heads - k.head);
  k.b = bi;
  k.t = token - bi * tokens;
  return k;
}

__device__ __forceinline__ int64_t position_of(const QkRope& p, const Task& k) {
  if (!p.pos) return p.start + k.t;
  const int64_t i = k.b * p.pb + k.t * p.pt;
  return p.pos64 ? reinterpret_cast<const int64_t*>(p.pos)[i] : reinterpret_cast<const int32_t*>(p.pos)[i];
}

// cos and sin of an item's pairs (1, 0 behind the rotated part).  A position that the tables do not hold reads nothing.
template <int V>
__device__ __forceinline__ void load_angles(const QkRope& p, bool in, int64_t at, int pair, float (&c)[V], float (&s)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) c[e] = 1.0f, s[e] = 0.0f;
  if (pair < 0 || !in) return;
  Chunk<WFB_F32, V> x, y;
  x.load(p.cos, at * (p.rotary / 2) + pair);
  y.load(p.sin, at * (p.rotary / 2) + pair);
#pragma unroll
  for (int e = 0; e < V; ++e) c[e] = x.get(e), s[e] = y.get(e);
}

// Forward, both sides' tasks in one range, a token's queries before its keys.  655k heads of 128 in bf16 (16384 tokens, 32/8
// heads) 66 us, 5.1 TB/s; a copy of the same bytes takes 70.  While loads were
// converted as they came: 94.
template <int DT, int V, int L, int IT>
__global__ __launch_bounds__(kThreads) void qk_rope_kernel(QkRope p, uint32_t tasks) {
  const int lane = threadIdx.x % L;
  const uint32_t i = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  const bool live = i < tasks;
  const uint32_t cq = (uint32_t)(p.side[0].heads + kHeads - 1) / kHeads, ck = (uint32_t)(p.side[1].heads + kHeads - 1) / kHeads;
  Task k = task_of(live ? i : 0, cq + ck, INT32_MAX, (uint32_t)p.t);
  const bool keys = (uint32_t)k.head >= cq * kHeads;
  const HeadRows sd = keys ? p.side[1] : p.side[0];
  k.head -= keys ? (int)cq * kHeads : 0;
  k.count = min(kHeads, sd.heads - k.head);
  const int D = p.head_dim, items = D / (2 * V);
  const int64_t at = position_of(p, k);
  const bool in = at >= 0 && at < p.rope_len, lost = p.rotary > 0 && !in;
  Chunk<DT, V> xa[IT][kHeads], xb[IT][kHeads];
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
      xa[it][h].zero();
      xb[it][h].zero();
      if (on[it] && h < k.count) {
        xa[it][h].load(sd.x, row + h * sd.xh + ea[it]);
        xb[it][h].load(sd.x, row + h * sd.xh + eb[it]);
      }
    }
  }
  float w[IT][2 * V], c[IT][V], s[IT][V];
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    load_angles<V>(p, in, at, on[it] ? pair[it] : -1, c[it], s[it]);
    item_weight<V>(sd, on[it], ea[it], eb[it], w[it]);
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    float r = 1.0f;
    if (sd.w) {  // (the lanes of a row agree)
      float ss = 0.0f;
#pragma unroll
      for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          ss = __builtin_fmaf(xa[it][h].get(e), xa[it][h].get(e), ss);
          ss = __builtin_fmaf(xb[it][h].get(e), xb[it][h].get(e), ss);
        }
      r = inverse_root(row_sum<L>(ss) / (float)D + p.eps);
    }
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      if (!on[it] || h >= k.count) continue;
      float y[2 * V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        y[e] = xa[it][h].get(e) * r * w[it][e];
        y[V + e] = xb[it][h].get(e) * r * w[it][V + e];
      }
      if (pair[it] >= 0) turn<V>(y, c[it], s[it], p.interleaved);
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

// Backward: the workgroups walk the queries' tasks, then the keys', and leave each side's part of the weight's gradient.
// 205k heads of 128 in bf16 (8192 tokens, 20/5 heads): 38 us for 157 MB (4.1 TB/s), and 4 for the sum over the groups.
// With the forward pass 64 us; 94 while a thread held both sides' sums and converted its loads as they came.
template <int DT, int V, int L, int IT>
__global__ __launch_bounds__(kThreads) void qk_rope_grad_kernel(QkRope p, float* __restrict__ part) {
  __shared__ float red[kThreads / L][2 * V * IT * L];
  constexpr int G = kThreads / L;
  const int lane = threadIdx.x % L, grp = threadIdx.x / L;
  const int D = p.head_dim, items = D / (2 * V);
  int ea[IT], eb[IT], pair[IT];
#pragma unroll
  for (int it = 0; it < IT; ++it) item_place<V>(p, min(lane + L * it, items - 1), ea[it], eb[it], pair[it]);

#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const HeadRows sd = side ? p.side[1] : p.side[0];
    const uint32_t chunks = (uint32_t)(sd.heads + kHeads - 1) / kHeads, tasks = (uint32_t)(p.batch * p.t) * chunks;
    float acc[IT][2 * V], w[IT][2 * V];
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      item_weight<V>(sd, true, ea[it], eb[it], w[it]);
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) acc[it][e] = 0.0f;
    }
    // every group of the workgroup takes the same number of turns, so that the lanes of a wave stay together
    for (uint32_t i0 = blockIdx.x * G; i0 < tasks; i0 += gridDim.x * G) {
      const bool live = i0 + grp < tasks;
      const Task k = task_of(live ? i0 + grp : 0, chunks, sd.heads, (uint32_t)p.t);
      const int64_t at = position_of(p, k);
      const bool in = at >= 0 && at < p.rope_len, lost = p.rotary > 0 && !in;
      const int64_t row = k.b * sd.xb + k.t * sd.xt + k.head * sd.xh, grow = k.b * sd.gb + k.t * sd.gt + k.head * sd.gh;
      Chunk<DT, V> xa[IT][kHeads], xb[IT][kHeads], ga[IT][kHeads], gb[IT][kHeads];
      float c[IT][V], s[IT][V];
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const bool on = live && lane + L * it < items;
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          ga[it][h].zero(), gb[it][h].zero(), xa[it][h].zero(), xb[it][h].zero();
          if (on && h < k.count) {
            ga[it][h].load(sd.g, grow + h * sd.gh + ea[it]);
            gb[it][h].load(sd.g, grow + h * sd.gh + eb[it]);
            if (sd.w) {
              xa[it][h].load(sd.x, row + h * sd.xh + ea[it]);
              xb[it][h].load(sd.x, row + h * sd.xh + eb[it]);
            }
          }
        }
        load_angles<V>(p, in, at, on ? pair[it] : -1, c[it], s[it]);
#pragma unroll
        for (int e = 0; e < V; ++e) s[it][e] = -s[it][e];  // turned back
      }
#pragma unroll
      for (int h = 0; h < kHeads; ++h) {
        float g[IT][2 * V], ss = 0.0f, sg = 0.0f;
#pragma unroll
        for (int it = 0; it < IT; ++it) {
#pragma unroll
          for (int e = 0; e < V; ++e) g[it][e] = ga[it][h].get(e), g[it][V + e] = gb[it][h].get(e);
          if (pair[it] >= 0) turn<V>(g[it], c[it], s[it], p.interleaved);
          if (lost) {
#pragma unroll
            for (int e = 0; e < 2 * V; ++e) g[it][e] = __builtin_nanf("");
          }
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float a = xa[it][h].get(e), b = xb[it][h].get(e);
            ss = __builtin_fmaf(a, a, __builtin_fmaf(b, b, ss));
            sg = __builtin_fmaf(g[it][e] * w[it][e], a, __builtin_fmaf(g[it][V + e] * w[it][V + e], b, sg));
          }
        }
        float r = 1.0f, m = 0.0f;
        if (sd.w) {
          r = inverse_root(row_sum<L>(ss) / (float)D + p.eps);
          m = r * (row_sum<L>(sg) / (float)D);
        }
#pragma unroll
        for (int it = 0; it < IT; ++it) {
          const bool on = live && lane + L * it < items && h < k.count;
          float y[2 * V];
          if (sd.w) {
#pragma unroll
            for (int e = 0; e < 2 * V; ++e) {
              const float n = (e < V ? xa[it][h].get(e) : xb[it][h].get(e - V)) * r;
              // (a row past the last one has x = 0, and with eps = 0 its n is NaN; one without a position adds its NaN)
              acc[it][e] = on ? __builtin_fmaf(g[it][e], n, acc[it][e]) : acc[it][e];
              y[e] = r * __builtin_fmaf(g[it][e], w[it][e], -(n * m));
            }
          } else {
#pragma unroll
            for (int e = 0; e < 2 * V; ++e) y[e] = g[it][e];
          }
          if (on && sd.out) {
            const int64_t o = ((k.b * p.t + k.t) * sd.heads + k.head + h) * D;
            store_chunk<DT, V>(sd.out, o + ea[it], &y[0]);
            store_chunk<DT, V>(sd.out, o + eb[it], &y[V]);
          }
        }
      }
    }
    if (!part) continue;
    if (side) __syncthreads();  // the first side's sums are read
#pragma unroll
    for (int it = 0; it < IT; ++it)
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) red[grp][(it * 2 * V + e) * L + lane] = acc[it][e];
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * V * IT * L; i += kThreads) {
      float u[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // (short chains: the sum's error grows with their length)
#pragma unroll
      for (int q = 0; q < G; ++q) u[q % 4] += red[q][i];
      const float v = (u[0] + u[1]) + (u[2] + u[3]);
      const int ln = i % L, e = i / L % (2 * V), it = i / L / (2 * V), j = ln + L * it;
      if (j >= items) continue;
      int a, b, pr;
      item_place<V>(p, j, a, b, pr);
      part[((int64_t)blockIdx.x * 2 + side) * D + (e < V ? a + e : b + e - V)] = v;
    }
  }
}

// Workgroups of the backward pass, three per CU: each leaves a row of partial sums for each weight, which the second launch
// adds up.
constexpr int kGradGroups = 768;

// The widest chunk that the sizes, strides and addresses allow: whole pairs on either side of the rotated part's end,
// chunks that start at multiples of their length in every row, and in the tables' rows.
int chunk_of(const QkRope& p, int dtype, bool grad) {
  const int esz = dtype == WFB_F32 ? 4 : 2;
  auto fits = [&](int v) {
    if (p.rotary % (2 * v) || (p.head_dim - p.rotary) % (2 * v)) return false;
    auto whole = [&](const void* q, int64_t a, int64_t b, int64_t c, int heads) {  // (a stride along one element never counts)
      return (uintptr_t)q % (v * esz) == 0 && (a % v == 0 || p.batch <= 1) && (b % v == 0 || p.t <= 1) &&
             (c % v == 0 || heads <= 1);
    };
    for (const HeadRows& s : p.side) {
      if (!whole(s.x, s.xb, s.xt, s.xh, s.heads) || !whole(s.out, 0, 0, 0, s.heads)) return false;
      if (grad && !whole(s.g, s.gb, s.gt, s.gh, s.heads)) return false;
      const int wv = v * (s.wdt == WFB_F32 ? 4 : 2);
      if (s.w && (uintptr_t)s.w % (wv < 16 ? wv : 16) != 0) return false;
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
  if (!grad) {
    const int64_t tasks = qk_tasks(p);
    const int64_t grid = (tasks + kThreads / L - 1) / (kThreads / L);
    hipLaunchKernelGGL((qk_rope_kernel<DT, V, L, IT>), dim3((unsigned)grid), dim3(kThreads), 0, s, p, (uint32_t)tasks);
  } else {
    hipLaunchKernelGGL((qk_rope_grad_kernel<DT, V, L, IT>), dim3((unsigned)groups), dim3(kThreads), 0, s, p, part);
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
    for (int u = 0; u < 8; ++u) v[u] = i + 16 * u < rows ? v[u] : 0.0f;
    acc += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
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
