// The int8 key/value cache: what its kernels share.
//
// A row is the head_dim elements of one token's key (after the rotary embedding) or value in one kv head.  It is held
// as int8 codes and one fp32 scale, m = max|x|, scale = m / 127, code = round_half_even(x * (127 / m)), each operation
// rounded to fp32, so the codes are reproducible bit for bit by any correctly rounded fp32 restatement.  Rows with
// m < 2^-100 hold scale 0 and codes 0 (127 / m would leave the range of fp32 below 2^-121), rows with a NaN or an
// infinity scale NaN and codes 0: such a row reads back as NaN, and so does whatever attends to it.
//
// Layout (cap, a multiple of 64, keys per sequence):
//   k        [batch, kv_heads, cap, D]         one key = D contiguous bytes
//   v        [batch, kv_heads, cap / 64, D, 64] blocks of 64 keys, transposed: the 16 or 32 elements x 64 keys that the
//            matrix cores take as the left operand of P V are contiguous, without a transposition on the way
//   k_scale, v_scale fp32 [batch, kv_heads, cap]
#pragma once

#include "wfb_common.h"

namespace wfb {

constexpr int kKvBlock = WFB_KV_I8_BLOCK;
constexpr float kKvTiny = 0x1p-100f;

// Where each sequence of a call writes and attends: sequence i adds tokens at positions first .. first + n - 1 of its
// cache.
struct KvSpan {
  const int64_t* start_dev;  // [batch] or null: start for all
  int64_t start;
  const int64_t* len_dev;    // [batch] or null: t for all
  int64_t t;                 // rows per sequence
  int64_t limit;             // positions below it may be used (cache capacity, rotary rows)
};

// False where a sequence's positions do not fit: nothing of it is written and its rows of a result are NaN.
__device__ __forceinline__ bool kv_span(const KvSpan& s, int b, int64_t& first, int& n) {
  first = s.start_dev ? s.start_dev[b] : s.start;
  const int64_t len = s.len_dev ? s.len_dev[b] : s.t;
  n = (int)len;
  return len >= 0 && len <= s.t && first >= 0 && first <= s.limit - len;
}

// Scale and factor of a row from its largest magnitude (as the bits of a non-negative float: an integer maximum keeps
// infinities and NaN above every finite value).
__device__ __forceinline__ void kv_scale(uint32_t mbits, float& scale, float& inv) {
  const float m = __uint_as_float(mbits);
  const bool some = m >= kKvTiny, finite = mbits < 0x7f800000u;
  scale = !finite ? __builtin_nanf("") : some ? __fdiv_rn(m, 127.0f) : 0.0f;
  inv = finite && some ? __fdiv_rn(127.0f, m) : 0.0f;
}

// round_half_even(x * inv) as the low byte; |x * inv| <= 127 (1 + 2^-22), and 0 for a row without codes (a NaN there
// would be clamped to -127 by the order of the operands)
__device__ __forceinline__ int kv_code(float x, float inv) {
  const float c = inv == 0.0f ? 0.0f : __fmul_rn(x, inv);
  return (int)__builtin_rintf(fminf(fmaxf(c, -127.0f), 127.0f));
}

hipError_t launch_kv_write_i8(int dt, int d, const void* kn, int64_t ldk, const void* vn, int64_t ldv, const float* rc,
                              const float* rs, int64_t turn, const wfb_kv_i8& c, const KvSpan& sp, int b, int hkv,
                              hipStream_t s);
hipError_t launch_kv_read_i8(int dt, int d, const wfb_kv_i8& c, const int64_t* start_dev, int64_t start, int b,
                             int64_t count, int hkv, void* k, void* v, hipStream_t s);

// One attention call.  Rows of q and out: row b * t + i is token i of sequence b.
struct KvAttn {
  const void* q;
  int64_t ldq;
  const void* kn;
  int64_t ldk;
  const void* vn;
  int64_t ldv;
  const float* rc;
  const float* rs;
  wfb_kv_i8 own, pre;  // pre: the shared prefix, read by every sequence before its own keys
  int64_t npre;        // keys of the prefix, 0 for none
  KvSpan span;
  int b, t, hq, hkv, d, dt;
  float scale;
  void* out;
  int64_t ldo;
  float* ws;
};
int64_t kv_attn_workspace_floats(int64_t batch, int64_t t, int64_t hq, int64_t hkv, int64_t d, int64_t cap,
                                 int64_t npre);
hipError_t launch_kv_attention(const KvAttn& a, hipStream_t s);

}  // namespace wfb
