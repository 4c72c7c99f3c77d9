// C-ABI entry points of the attention of sequences that share a prefix.
// Argument checks are HIP-free, as in capi.cpp.
#include "capi_checks.h"

namespace dsa {

// paged_prefix.hip
bool paged_prefix_launchable(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                             int64_t max_blocks, int64_t page);
size_t paged_prefix_workspace_bytes(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                                    int64_t max_blocks, int64_t page, int64_t min_tokens);
int paged_prefix_run(const void* query, const void* query_rope, const void* key, const void* key_rope,
                     const void* value, void* out, float* smax, float* ssum, const int32_t* act_q,
                     const int32_t* act_k, const int32_t* table, const int32_t* ids, const int32_t* shared,
                     int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, int64_t num_blocks, int64_t page,
                     int64_t max_blocks, int32_t mode, int64_t pre_tokens, int64_t next_tokens, int64_t min_tokens,
                     int32_t dtype, float scale, int32_t return_lse, void* workspace, hipStream_t stream);

}  // namespace dsa

using namespace dsa;

extern "C" {

size_t dsa_paged_prefix_attn_workspace_size(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d,
                                            int32_t latent, int64_t max_blocks, int64_t page_size) {
  return dsa_paged_prefix_attn_workspace_bytes(batch, s1, n1, n2, d, latent, max_blocks, page_size, 0);
}

size_t dsa_paged_prefix_attn_workspace_bytes(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d,
                                             int32_t latent, int64_t max_blocks, int64_t page_size,
                                             int64_t min_tokens) {
  if (!paged_attn_sizes_ok(batch, s1, n1, n2, d, latent != 0, max_blocks, page_size) ||
      !paged_prefix_launchable(batch, s1, n1, n2, d, latent != 0, max_blocks, page_size))
    return 0;
  return paged_prefix_workspace_bytes(batch, s1, n1, n2, d, latent != 0, max_blocks, page_size, min_tokens);
}

int dsa_paged_prefix_attn(const void* query, const void* query_rope, const void* key, const void* key_rope,
                          const void* value, void* attention_out, float* softmax_max, float* softmax_sum,
                          const int32_t* actual_seq_q, const int32_t* actual_seq_kv, const int32_t* block_table,
                          const int32_t* prefix_groups, const int32_t* prefix_lengths, int64_t batch, int64_t s1,
                          int64_t n1, int64_t n2, int64_t d, int64_t d_rope, int64_t num_blocks, int64_t page_size,
                          int64_t max_blocks, int32_t sparse_mode, int64_t pre_tokens, int64_t next_tokens,
                          int64_t min_tokens, int32_t dtype, float scale_value, int32_t return_lse, void* workspace,
                          size_t workspace_bytes, void* stream) {
  clear_error();
  const bool latent = value == nullptr;
  DSA_CHECK_ARG(prefix_groups && prefix_lengths, "null tensor pointer");
  int st = check_paged_attn(query, query_rope, key, key_rope, value, attention_out, softmax_max, softmax_sum,
                            actual_seq_kv, block_table, batch, s1, n1, n2, d, d_rope, num_blocks, page_size, max_blocks,
                            sparse_mode, dtype, return_lse);
  if (st != DSA_OK) return st;
  DSA_CHECK_SUPPORTED(paged_prefix_launchable(batch, s1, n1, n2, d, latent, max_blocks, page_size),
                      "too many query rows, or too many for so wide a block table");
  st = check_workspace(workspace, workspace_bytes,
                       paged_prefix_workspace_bytes(batch, s1, n1, n2, d, latent, max_blocks, page_size, min_tokens));
  if (st != DSA_OK) return st;
  DSA_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
  return paged_prefix_run(query, query_rope, key, key_rope, value, attention_out, softmax_max, softmax_sum,
                          actual_seq_q, actual_seq_kv, block_table, prefix_groups, prefix_lengths, batch, s1, n1, n2, d,
                          num_blocks, page_size, max_blocks, sparse_mode, pre_tokens, next_tokens, min_tokens, dtype,
                          scale_value, return_lse, workspace, (hipStream_t)stream);
}

}  // extern "C"
