// Checks of arguments that the entry points of the operators around paged
// caches share (HIP-free, as in capi.cpp).
#pragma once

#include "common.h"

namespace dsa {

// paged_attn.hip
bool paged_attn_launchable(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                           int64_t max_blocks, int64_t page);

// a * b <= lim without overflow, for non-negative factors
static bool within(int64_t a, int64_t b, int64_t lim) {
  int64_t r;
  return a >= 0 && b >= 0 && !__builtin_mul_overflow(a, b, &r) && r <= lim;
}

static int check_pages(int64_t pages, int64_t page, int64_t max_blocks) {
  DSA_CHECK_ARG(page >= 1 && page <= (1 << 20), "page (block) size must be in [1, 2^20]");
  DSA_CHECK_ARG(pages >= 1 && max_blocks >= 1, "the cache and the block table need at least one block");
  DSA_CHECK_ARG(max_blocks <= (1 << 20) && within(max_blocks, page, 65535ll * 1024),
                "max_blocks * page size must be <= 67107840 (max_blocks <= 2^20)");
  DSA_CHECK_ARG(within(pages, page, (1ll << 31) - 1), "the cache must have fewer than 2^31 rows");
  return DSA_OK;
}

static int check_workspace(const void* workspace, size_t bytes, size_t need) {
  if (need && (workspace == nullptr || bytes < need)) {
    set_error("workspace of %zu bytes required, %zu given", need, bytes);
    return DSA_ERR_WORKSPACE;
  }
  return DSA_OK;
}

constexpr int64_t kMaxTableTokens = 1ll << 35;  // of a block table: the kernels count its 32-token tiles in 32 bits

static bool paged_attn_sizes_ok(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                                int64_t max_blocks, int64_t page) {
  return batch >= 1 && batch <= (1 << 24) && s1 >= 1 && n2 >= 1 && n1 >= n2 && n1 % n2 == 0 &&
         within(s1, n1, 1ll << 24) && within(batch * s1, n1, (1ll << 31) - 1) &&
         (latent ? n2 == 1 && (d == 128 || d == 256 || d == 512) : d == 64 || d == 128 || d == 256) &&
         page >= 1 && page <= (1 << 20) && max_blocks >= 1 && max_blocks <= (1 << 20) &&
         within(max_blocks, page, 65535ll * 1024) && within(batch, max_blocks * page, kMaxTableTokens) &&
         paged_attn_launchable(batch, s1, n1, n2, d, latent, max_blocks, page);
}

// the arguments that every attention over pages has
static int check_paged_attn(const void* query, const void* query_rope, const void* key, const void* key_rope,
                            const void* value, const void* attention_out, const float* softmax_max,
                            const float* softmax_sum, const int32_t* actual_seq_kv, const int32_t* block_table,
                            int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, int64_t d_rope,
                            int64_t num_blocks, int64_t page_size, int64_t max_blocks, int32_t sparse_mode,
                            int32_t dtype, int32_t return_lse) {
  const bool latent = value == nullptr;
  DSA_CHECK_ARG(query && key && attention_out && actual_seq_kv && block_table, "null tensor pointer");
  DSA_CHECK_ARG((softmax_max == nullptr) == (softmax_sum == nullptr) && (!return_lse || softmax_max),
                "softmax_max and softmax_sum must be both provided (return_softmax_lse) or both omitted");
  DSA_CHECK_SUPPORTED(dtype == DSA_DTYPE_BF16 || dtype == DSA_DTYPE_FP16, "query dtype must be bfloat16 or float16");
  DSA_CHECK_SUPPORTED(sparse_mode == 0 || sparse_mode == 3, "Only sparse_mode 0 (full) / 3 (rightDownCausal) supported");
  if (latent) {
    DSA_CHECK_ARG(query_rope && key_rope, "the latent form (no value) needs query_rope and key_rope");
    DSA_CHECK_SUPPORTED(d == 128 || d == 256 || d == 512, "D must be one of (128, 256, 512), got %lld", (long long)d);
    DSA_CHECK_SUPPORTED(d_rope == 64, "rope dim must be 64, got %lld", (long long)d_rope);
    DSA_CHECK_SUPPORTED(n2 == 1, "the latent form has one key head, got %lld", (long long)n2);
  } else {
    DSA_CHECK_ARG(!query_rope && !key_rope && d_rope == 0, "the grouped form (with value) takes no rope parts");
    DSA_CHECK_SUPPORTED(d == 64 || d == 128 || d == 256, "D must be one of (64, 128, 256), got %lld", (long long)d);
  }
  DSA_CHECK_ARG(n1 >= 1 && n2 >= 1 && n1 % n2 == 0, "query N1 must be divisible by key N2");
  DSA_CHECK_ARG(batch >= 1 && batch <= (1 << 24) && s1 >= 1, "batch must be in [1, 2^24], S1 at least 1");
  DSA_CHECK_ARG(within(s1, n1, 1ll << 24) && within(batch * s1, n1, (1ll << 31) - 1), "too many query rows");
  int st = check_pages(num_blocks, page_size, max_blocks);
  if (st != DSA_OK) return st;
  DSA_CHECK_SUPPORTED(within(batch, max_blocks * page_size, kMaxTableTokens),
                      "batch * max_blocks * page size must be <= 2^35");
  DSA_CHECK_SUPPORTED(paged_attn_launchable(batch, s1, n1, n2, d, latent, max_blocks, page_size),
                      "too many query rows for one launch");
  // 16-byte loads of rows
  DSA_CHECK_ARG((((uintptr_t)query | (uintptr_t)key | (uintptr_t)value | (uintptr_t)query_rope | (uintptr_t)key_rope |
                  (uintptr_t)attention_out) & 15) == 0, "tensors must be 16-byte aligned");
  return DSA_OK;
}

}  // namespace dsa
