// Host-side AddressSanitizer driver for the training step's entry points (built with the host-only ASan library by
// wrinklefree-monorepo_amd/_build.py build_asan; run by tests/test_asan_train_ops.py, no GPU needed): each call below must
// be refused with WFB_EINVAL and a message, without touching the fake device pointers it is given, or do host work only.
// Exit status 0 when every expectation held; ASan aborts the process on a memory error.
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include "wfbitnet.h"

static int g_fail = 0;
static void expect(bool ok, const char* what) {
  if (!ok) {
    std::fprintf(stderr, "FAILED: %s\n", what);
    ++g_fail;
  }
}

static void* fake(uintptr_t a) { return reinterpret_cast<void*>(a); }  // never dereferenced on the host

static void refused(int st, const char* what) {
  expect(st == WFB_EINVAL && std::strlen(wfb_last_error()) > 0, what);
}

int main() {
  auto* x = static_cast<float*>(fake(0x1000));
  auto* q = static_cast<uint8_t*>(fake(0x2000));
  auto* c = static_cast<int8_t*>(fake(0x3000));
  auto* d = static_cast<double*>(fake(0x4000));
  refused(wfb_pack_gated(x, x, 7, 64, 256, x, q, d, nullptr), "pack dtype");
  refused(wfb_pack_gated(x, nullptr, WFB_F32, 64, 256, x, q, d, nullptr), "pack null");
  refused(wfb_gated_i2s(q, 64, 200, c, 4, 256, x, x, WFB_ACT_SILU, x, WFB_F32, x, nullptr), "K");
  refused(wfb_gated_i2s(q, 64, 256, c, 4, 256, x, x, 9, x, WFB_F32, x, nullptr), "activation");
  refused(wfb_gated_i2s(q, 64, 256, c, 4, 128, x, x, WFB_ACT_SILU, x, WFB_F32, nullptr, nullptr), "stride");
  int64_t n = 0;
  for (int64_t m : {1, 63, 64, 65, 4096, 1048575})
    for (int64_t f : {1, 64, 65, 14336, 524287})
      for (int wants = 1; wants < 4; ++wants)
        for (int dt : {WFB_F32, WFB_BF16})
          expect(wfb_gated_grad_workspace(m, f, 4097, dt, wants & 1, dt, wants & 2, &n) == WFB_OK && n > 0, "workspace");
  refused(wfb_gated_grad_workspace(-1, 1, 1, WFB_F32, 1, WFB_F32, 1, &n), "workspace sizes");
  refused(wfb_gated_grad(x, x, WFB_F32, 63, 4, 64, WFB_ACT_SILU, q, 256, 256, x, c, 256, x, x, WFB_F32, x, WFB_F32, x, nullptr),
          "gradient stride");
  refused(wfb_gated_grad(x, x, WFB_F32, 64, 0, 64, WFB_ACT_SILU, q, 256, 256, x, c, 256, x, x, WFB_F32, x, WFB_F32, x, nullptr),
          "no rows");

  wfb_heads h{x, 512, 128, 64, x, 512, 128, 64, nullptr, 0, x, nullptr, 2};
  wfb_rope r{x, x, 16, 64, 0, nullptr, 0, 0, 0, 0};
  refused(wfb_qk_norm_rope(&h, &h, nullptr, WFB_F32, 1, 4, 64, 1e-6f, nullptr), "null rope");
  refused(wfb_qk_norm_rope(&h, &h, &r, WFB_F32, 1, 4, 300, 1e-6f, nullptr), "head_dim");
  refused(wfb_qk_norm_rope(&h, &h, &r, WFB_F32, 1, 17, 64, 1e-6f, nullptr), "positions");
  wfb_heads none = h;
  none.x = nullptr;
  refused(wfb_qk_norm_rope(&h, &none, &r, WFB_F32, 1, 4, 64, 1e-6f, nullptr), "null heads");
  wfb_heads loose = h;
  loose.grad_weight = x;
  refused(wfb_qk_norm_rope_grad(&h, &loose, &r, WFB_F32, 1, 4, 64, 1e-6f, x, nullptr), "gradient without a weight");
  expect(wfb_qk_norm_rope(&h, &h, &r, WFB_F32, 0, 4, 64, 1e-6f, nullptr) == WFB_OK, "no batch");
  expect(wfb_qk_norm_rope_grad_workspace(2, 3, 4, 5, 64, &n) == WFB_OK && n > 0, "rope workspace");
  refused(wfb_qk_norm_rope_grad_workspace(2, 3, 4, 5, 64, nullptr), "rope workspace null");

  std::vector<float> cos(6 * 3), sin(6 * 3);
  const double inv[3] = {1.0, 0.1, 0.01};
  expect(wfb_rope_tables_scaled(inv, 3, 1.0, 6, cos.data(), sin.data()) == WFB_OK && cos[0] == 1.0f && sin[0] == 0.0f, "tables");
  refused(wfb_rope_tables_scaled(inv, 0, 1.0, 6, cos.data(), sin.data()), "no pairs");
  refused(wfb_rope_tables_scaled(nullptr, 3, 1.0, 6, cos.data(), sin.data()), "null frequencies");

  std::vector<wfb_adamw_tensor> t(200, wfb_adamw_tensor{x, x, 300});
  auto step = [&](int64_t elements, int bits, int64_t at) {
    return wfb_adamw_step(t.data(), (int64_t)t.size(), WFB_F32, WFB_F32, x, x, bits == 8 ? x : nullptr, bits == 8 ? x : nullptr,
                          elements, bits, 1e-3, 0.9, 0.99, 1e-8, 0.0, at, nullptr, nullptr, nullptr, nullptr);
  };
  refused(step(512 * 199, 32, 1), "the last tensor leaves the state");
  refused(step(512 * 201, 32, 1), "the state is larger");
  refused(step(512 * 200, 16, 1), "bits");
  refused(step(512 * 200, 8, 0), "step");
  t[150].p = nullptr;
  refused(step(512 * 200, 8, 1), "null tensor");
  expect(wfb_adamw_step(nullptr, 0, WFB_F32, WFB_F32, x, x, nullptr, nullptr, 256, 32, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, nullptr,
                        nullptr, nullptr, nullptr) == WFB_OK, "no tensors");
  refused(wfb_adamw_values(x, x, x, nullptr, 256, x, x, nullptr), "null scale");
  std::printf("train_ops: %d failures\n", g_fail);
  return g_fail != 0;
}
