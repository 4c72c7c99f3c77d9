// Host-side sanitizer check of the paged decoding entry points (test
// infrastructure), in the manner of capi_check.cpp: every call from a small
// valid configuration with one argument at a time at an extreme value or NULL,
// on a machine without a GPU, where a call that passes validation fails at
// its first HIP call.  The few functions of capi.cpp that these sources use
// are defined here, so that only they are built with the sanitizers.
#include <hip/hip_runtime_api.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <functional>
#include <string>
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

typedef std::function<int(const std::vector<const void*>&, const std::vector<int64_t>&)> Call;

void one(const char* name, const std::string& what, int st, bool null) {
  ++g_cases;
  std::string bad;
  if (st < DSA_OK || st > DSA_ERR_WORKSPACE) bad = "status";
  if (st != DSA_OK && !dsa::g_err[0]) bad = "no message";
  if (null && st != DSA_ERR_INVALID && st != DSA_ERR_WORKSPACE) bad = "NULL not rejected";
  if (!bad.empty()) {
    ++g_fail;
    fprintf(stderr, "FAIL %s %s: %s (%d)\n", name, what.c_str(), bad.c_str(), st);
  }
}

void sweep(const char* name, int nptr, const std::vector<int>& optional, const std::vector<int64_t>& ints,
           const Call& call) {
  std::vector<const void*> p;
  for (int i = 0; i < nptr; ++i) p.push_back((const void*)(uintptr_t)(0x10000 + 0x1000 * i));
  one(name, "baseline", call(p, ints), false);
  for (size_t i = 0; i < ints.size(); ++i)
    for (int64_t x : kExtremes) {
      auto v = ints;
      v[i] = x;
      one(name, "int " + std::to_string(i) + " = " + std::to_string(x), call(p, v), false);
    }
  for (int i = 0; i < nptr; ++i) {
    auto q = p;
    q[i] = nullptr;
    bool opt = false;
    for (int o : optional) opt |= o == i;
    one(name, "ptr " + std::to_string(i) + " = NULL", call(q, ints), !opt);
  }
}

}  // namespace

int main() {
  int n = 0;
  if (hipGetDeviceCount(&n) == hipSuccess && n > 0) {
    printf("SKIP a GPU is present\n");
    return 0;
  }
  typedef const std::vector<const void*>& Ps;
  typedef const std::vector<int64_t>& Is;
  sweep("rope", 6, {2, 3}, {64, 64, 64, 64, 64, 64, 2, 64, 0, 64, 64, 64, 64, 64, 64, 1, 64, 0, 0, 1, 2, 3, 32, 0, 0, 0},
        [](Ps p, Is v) {
          return dsa_rope(p[0], (void*)p[1], v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], p[2], (void*)p[3],
                          v[9], v[10], v[11], v[12], v[13], v[14], v[15], v[16], v[17], p[4], (int32_t)v[18],
                          (int32_t)v[19], (const double*)p[5], v[20], v[21], v[22], (int32_t)v[23], (int32_t)v[24],
                          (int32_t)v[25], 1.f, nullptr);
        });
  // lists of two caches, in host memory
  static const void* rows[2] = {(void*)0x90000, (void*)0x91000};
  static void* caches[2] = {(void*)0x80000, (void*)0x81000};
  sweep("paged_cache_write", 3, {2}, {128, 64, 256, 128, 2, 2, 3, 6, 4, 8, 16, 0}, [](Ps p, Is v) {
    const int64_t bytes[2] = {v[0], 64}, sb[2] = {v[2], 256}, st[2] = {v[3], 64};
    (void)v[1];
    return dsa_paged_cache_write(v[4] > 2 ? 2 : v[4], rows, caches, bytes, sb, st, (const int32_t*)p[0],
                                 (const int32_t*)p[1], (const int32_t*)p[2], v[5], v[6], v[7], v[8], v[9], v[10],
                                 (int32_t)v[11], nullptr);
  });
  sweep("paged_cache_fork", 8, {3}, {128, 2, 2, 3, 4, 4, 8, 16, 1, 1 << 20}, [](Ps p, Is v) {
    const int64_t bytes[2] = {v[0], 64};
    return dsa_paged_cache_fork(v[1] > 2 ? 2 : v[1], caches, bytes, (const int32_t*)p[0], (const int32_t*)p[1],
                                (const int32_t*)p[2], (const int32_t*)p[3], (int32_t*)p[4], (int32_t*)p[5],
                                (int32_t*)p[6], v[2], v[3], v[4], v[5], v[6], v[7], v[8], (void*)p[7], (size_t)v[9],
                                nullptr);
  });
  sweep("paged_cache_compact", 6, {}, {128, 2, 2, 4, 8, 16, 1 << 20}, [](Ps p, Is v) {
    const int64_t bytes[2] = {v[0], 64};
    return dsa_paged_cache_compact(v[1] > 2 ? 2 : v[1], caches, bytes, (const int32_t*)p[0], (const int32_t*)p[1],
                                   (int32_t*)p[2], (int32_t*)p[3], (int32_t*)p[4], v[2], v[3], v[4], v[5],
                                   (void*)p[5], (size_t)v[6], nullptr);
  });
  for (int latent = 0; latent < 2; ++latent) {
    // query, query_rope, key, key_rope, value, out, max, sum, lengths (q, kv), table, workspace
    std::vector<int> opt = {8};  // and those that the form does not take
    if (latent) opt.push_back(4);
    else opt.insert(opt.end(), {1, 3});
    sweep(latent ? "paged_attn latent" : "paged_attn grouped", 12, opt,
          {2, 1, 8, latent ? 1 : 2, latent ? 512 : 128, latent ? 64 : 0, 8, 16, 4, 3, 1ll << 62, 1ll << 62, 0, 1,
           1ll << 40},
          [latent](Ps p, Is v) {
            return dsa_paged_attn(p[0], latent ? p[1] : nullptr, p[2], latent ? p[3] : nullptr,
                                  latent ? nullptr : p[4], (void*)p[5], (float*)p[6], (float*)p[7],
                                  (const int32_t*)p[8], (const int32_t*)p[9], (const int32_t*)p[10], v[0], v[1], v[2],
                                  v[3], v[4], v[5], v[6], v[7], v[8], (int32_t)v[9], v[10], v[11], (int32_t)v[12],
                                  0.1f, (int32_t)v[13], (void*)p[11], (size_t)v[14], nullptr);
          });
  }
  const std::vector<int64_t> sizes = {2, 1, 8, 2, 128, 0, 4, 16};
  for (size_t i = 0; i < sizes.size(); ++i)
    for (int64_t x : kExtremes) {
      auto v = sizes;
      v[i] = x;
      ++g_cases;
      (void)dsa_paged_attn_workspace_size(v[0], v[1], v[2], v[3], v[4], (int32_t)v[5], v[6], v[7]);
      (void)dsa_paged_cache_fork_workspace_size(v[0], v[1], v[2]);
      (void)dsa_paged_cache_compact_workspace_size(v[0]);
    }
  printf("%s %d cases, %d failures\n", g_fail ? "FAILED" : "OK", g_cases, g_fail);
  return g_fail != 0;
}
