// Host-side sanitizer check of the entry points that serve requests of many
// lengths (test infrastructure), in the manner of capi_check_decode.cpp: every
// call from a small valid configuration with one or two integers at a time at
// an extreme value, or one pointer NULL, on a machine without a GPU.
#include <hip/hip_runtime_api.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <functional>
#include <set>
#include <vector>

#include "dsa_capi.h"

namespace dsa {
static char g_err[512] = "";
void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}
void clear_error() { g_err[0] = '\0'; }
int hip_fail(hipError_t e, const char* what) {
  set_error("HIP error in %s: %s", what, hipGetErrorString(e));
  return DSA_ERR_HIP;
}
int device_cu_count() { return 256; }
int test_flags() { return 0; }
}  // namespace dsa

namespace {

const int64_t kExtremes[] = {-1, 0, 1, 3, 65, 4097, (1ll << 24) + 1, (1ll << 31) - 1, 1ll << 31, 1ll << 40, 1ll << 62,
                             INT64_MAX, INT64_MIN};
int g_cases = 0, g_fail = 0;

typedef const std::vector<const void*>& Ps;
typedef const std::vector<int64_t>& Is;

void expect(bool ok, const char* name, const char* what, int st, long long i, long long j) {
  ++g_cases;
  if (ok) return;
  ++g_fail;
  fprintf(stderr, "FAIL %s %s %lld %lld (%d)\n", name, what, i, j, st);
}

void sweep(const char* name, int nptr, const std::set<int>& optional, const std::vector<int64_t>& ints,
           const std::function<int(Ps, Is)>& call) {
  std::vector<const void*> p;
  for (int i = 0; i < nptr; ++i) p.push_back((const void*)(uintptr_t)(0x10000 + 0x1000 * i));
  auto sound = [](int st) { return st >= DSA_OK && st <= DSA_ERR_WORKSPACE && (st == DSA_OK || dsa::g_err[0]); };
  int st = call(p, ints);
  expect(st == DSA_OK || st == DSA_ERR_HIP, name, "baseline", st, 0, 0);
  for (size_t i = 0; i < ints.size(); ++i)
    for (size_t j = i; j < ints.size(); ++j)
      for (int64_t x : kExtremes) {
        auto v = ints;
        v[i] = v[j] = x;
        st = call(p, v);
        expect(sound(st), name, "integers", st, (long long)(i * 100 + j), (long long)x);
      }
  for (int i = 0; i < nptr; ++i) {
    auto q = p;
    q[i] = nullptr;
    st = call(q, ints);
    expect(sound(st) && (optional.count(i) || st == DSA_ERR_INVALID || st == DSA_ERR_WORKSPACE), name, "NULL", st, i, 0);
  }
}

}  // namespace

int main() {
  int n = 0;
  if (hipGetDeviceCount(&n) == hipSuccess && n > 0) {
    printf("SKIP a GPU is present\n");
    return 0;
  }
  static int64_t sections[4];
  sweep("rope_axes", 6, {2, 3},
        {64, 64, 64, 64, 64, 64, 2, 64, 0, 64, 64, 64, 64, 64, 64, 1, 64, 0, 0, 1, 2, 3, 32, 3, 6, 5, 5, 0, 0, 0, 0},
        [](Ps p, Is v) {
          for (int i = 0; i < 4; ++i) sections[i] = i < 3 ? v[24 + i] : 0;
          return dsa_rope_axes(p[0], (void*)p[1], v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], p[2],
                               (void*)p[3], v[9], v[10], v[11], v[12], v[13], v[14], v[15], v[16], v[17], p[4],
                               (int32_t)v[18], (int32_t)v[19], (const double*)p[5], v[20], v[21], v[22], (int32_t)v[23],
                               sections, (int32_t)v[27], (int32_t)v[28], (int32_t)v[29], (int32_t)v[30], 1.f, nullptr);
        });
  sweep("paged_cache_plan", 11, {}, {4, 4, 16, 16, 8, 1 << 20}, [](Ps p, Is v) {
    return dsa_paged_cache_plan((const int32_t*)p[0], (const int32_t*)p[1], (const int32_t*)p[2], (const int32_t*)p[3],
                                (int32_t*)p[4], (int32_t*)p[5], (int32_t*)p[6], (int32_t*)p[7], (int32_t*)p[8],
                                (int32_t*)p[9], v[0], v[1], v[2], v[3], v[4], (void*)p[10], (size_t)v[5], nullptr);
  });
  static const void* rows[2] = {(void*)0x90000, (void*)0x91000};
  static void* caches[2] = {(void*)0x80000, (void*)0x81000};
  sweep("paged_cache_write_slots", 1, {}, {128, 256, 128, 2, 2, 3, 8, 16}, [](Ps p, Is v) {
    const int64_t bytes[2] = {v[0], 64}, sb[2] = {v[1], 256}, st[2] = {v[2], 64};
    return dsa_paged_cache_write_slots(v[3] > 2 ? 2 : v[3], rows, caches, bytes, sb, st, (const int32_t*)p[0], v[4],
                                       v[5], v[6], v[7], nullptr);
  });
  sweep("paged_cache_prefixes", 4, {}, {4, 4, 16, 1}, [](Ps p, Is v) {
    return dsa_paged_cache_prefixes((const int32_t*)p[0], (const int32_t*)p[1], (int32_t*)p[2], (int32_t*)p[3], v[0],
                                    v[1], v[2], v[3], nullptr);
  });
  for (int latent = 0; latent < 2; ++latent) {
    // query, query_rope, key, key_rope, value, out, max, sum, lengths (q, kv), table, groups, shared, workspace
    std::set<int> opt = {8};  // and those that the form does not take
    if (latent) opt.insert(4);
    else opt.insert({1, 3});
    sweep(latent ? "paged_prefix_attn latent" : "paged_prefix_attn grouped", 14, opt,
          {2, 1, 8, latent ? 1 : 2, latent ? 512 : 128, latent ? 64 : 0, 8, 16, 4, 3, 1ll << 62, 1ll << 62, -1, 0,
           1, 1ll << 40},
          [latent](Ps p, Is v) {
            return dsa_paged_prefix_attn(p[0], latent ? p[1] : nullptr, p[2], latent ? p[3] : nullptr,
                                         latent ? nullptr : p[4], (void*)p[5], (float*)p[6], (float*)p[7],
                                         (const int32_t*)p[8], (const int32_t*)p[9], (const int32_t*)p[10],
                                         (const int32_t*)p[11], (const int32_t*)p[12], v[0], v[1], v[2], v[3], v[4],
                                         v[5], v[6], v[7], v[8], (int32_t)v[9], v[10], v[11], v[12],
                                         (int32_t)v[13], 0.1f, (int32_t)v[14], (void*)p[13], (size_t)v[15], nullptr);
          });
  }
  for (int latent = 0; latent < 2; ++latent) {
    const std::vector<int64_t> sizes = {2, 1, 8, latent ? 1 : 2, latent ? 512 : 128, latent, 4, 16};
    for (size_t i = 0; i < sizes.size(); ++i)
      for (size_t j = i; j < sizes.size(); ++j)
        for (int64_t x : kExtremes) {
          auto v = sizes;
          v[i] = v[j] = x;
          ++g_cases;
          (void)dsa_paged_prefix_attn_workspace_size(v[0], v[1], v[2], v[3], v[4], (int32_t)v[5], v[6], v[7]);
          (void)dsa_paged_cache_plan_workspace_size(v[0], v[1]);
        }
  }
  printf("%s %d cases, %d failures\n", g_fail ? "FAILED" : "OK", g_cases, g_fail);
  return g_fail != 0;
}
