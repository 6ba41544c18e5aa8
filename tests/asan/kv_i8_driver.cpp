// Host-side AddressSanitizer driver for the entry points of the int8 key/value cache (built with the host-only ASan library
// by wrinklefree-monorepo_amd/_build.py build_asan; run by tests/test_asan_kv_i8.py, no GPU needed): each call below must
// be refused with WFB_EINVAL and a message, without touching the fake device pointers it is given.
// Exit status 0 when every expectation held; ASan aborts the process on a memory error.
#include <cstdint>
#include <cstdio>
#include <cstring>

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
  wfb_kv_i8 c{static_cast<int8_t*>(fake(0x2000)), x, static_cast<int8_t*>(fake(0x3000)), x, 128};
  wfb_kv_i8 odd = c;
  odd.cap = 100;
  wfb_kv_i8 none = c;
  none.v = nullptr;
  refused(wfb_kv_write_i8(x, 128, x, 128, WFB_BF16, nullptr, nullptr, 0, 0, nullptr, nullptr, 0, nullptr, 1, 1, 2, 64, nullptr),
          "null cache");
  refused(wfb_kv_write_i8(x, 128, x, 128, WFB_BF16, nullptr, nullptr, 0, 0, &odd, nullptr, 0, nullptr, 1, 1, 2, 64, nullptr),
          "cache capacity");
  refused(wfb_kv_write_i8(x, 128, x, 128, WFB_BF16, nullptr, nullptr, 0, 0, &none, nullptr, 0, nullptr, 1, 1, 2, 64, nullptr),
          "null cache pointer");
  refused(wfb_kv_write_i8(x, 128, x, 128, WFB_BF16, nullptr, nullptr, 0, 0, &c, nullptr, 128, nullptr, 1, 1, 2, 64, nullptr),
          "position outside the cache");
  refused(wfb_kv_write_i8(x, 128, x, 128, WFB_BF16, x, x, 10, 8, &c, nullptr, 0, nullptr, 1, 3, 2, 64, nullptr),
          "position outside the rotary tables");
  refused(wfb_kv_read_i8(&c, nullptr, 0, 1, -1, 2, 64, x, x, WFB_F32, nullptr), "negative count");
  refused(wfb_kv_read_i8(&c, nullptr, 0, 1, 1, 2, 64, x, x, WFB_F16, nullptr), "read dtype");
  int64_t n = 0;
  refused(wfb_gqa_attention_i8_workspace(1, 1, 9, 2, 64, 128, 0, &n), "heads");
  refused(wfb_gqa_attention_i8_workspace(1, 1, 8, 2, 64, 128, 0, nullptr), "null size");
  expect(wfb_gqa_attention_i8_workspace(3, 17, 8, 2, 64, 131072, 5000, &n) == WFB_OK && n > 0, "workspace of a split call");
  refused(wfb_gqa_attention_i8(x, 512, x, 128, x, 128, WFB_BF16, nullptr, nullptr, 0, &c, nullptr, 0, nullptr, nullptr, 4, 1, 1,
                               8, 2, 64, 0.125f, x, 512, x, nullptr),
          "prefix length without a prefix");
  refused(wfb_gqa_attention_i8(x, 512, x, 128, x, 128, WFB_BF16, nullptr, nullptr, 0, &c, nullptr, 0, nullptr, &c, 129, 1, 1,
                               8, 2, 64, 0.125f, x, 512, x, nullptr),
          "prefix past its capacity");
  refused(wfb_gqa_attention_i8(x, 500, x, 128, x, 128, WFB_BF16, nullptr, nullptr, 0, &c, nullptr, 0, nullptr, nullptr, 0, 1, 1,
                               8, 2, 64, 0.125f, x, 512, x, nullptr),
          "query stride");
  std::printf("kv_i8: %d failures\n", g_fail);
  return g_fail != 0;
}
