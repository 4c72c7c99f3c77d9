// C-ABI entry points of the paged decoding operators: rotary positions, the
// pages of a cache, and attention over them.  Argument checks are HIP-free,
// as in capi.cpp.
#include "common.h"

namespace dsa {

// rope.hip
int rope_run(const void* const in[2], void* const out[2], const int64_t* const strides[2], const int64_t heads[2],
             const int64_t d[2], const int64_t start[2], int n, const void* positions, int32_t pos64,
             int32_t pos_per_seq, const double* inv_freq, int64_t tokens, int64_t s, int64_t rot, int32_t interleaved,
             int32_t inverse, int32_t dtype, float scale, hipStream_t stream);
// paged_cache.hip
int pc_write_run(int64_t n, const void* const* rows, void* const* caches, const int64_t* row_bytes,
                 const int64_t* row_sb, const int64_t* row_st, const int32_t* table, const int32_t* lens,
                 const int32_t* row_lengths, int64_t batch, int64_t s, int64_t tokens, int64_t max_blocks,
                 int64_t pages, int64_t page, int32_t layout, hipStream_t stream);
size_t pc_fork_workspace_bytes(int64_t rows, int64_t children, int64_t pages);
int pc_fork_run(int64_t n, void* const* caches, const int64_t* row_bytes, const int32_t* table, const int32_t* lens,
                const int32_t* refs, const int32_t* parents, int32_t* new_table, int32_t* new_lens,
                int32_t* new_refs, int64_t rows, int64_t children, int64_t max_blocks, int64_t new_blocks,
                int64_t pages, int64_t page, int64_t new_tokens, void* workspace, hipStream_t stream);
size_t pc_compact_workspace_bytes(int64_t pages);
int pc_compact_run(int64_t n, void* const* caches, const int64_t* row_bytes, const int32_t* table,
                   const int32_t* refs, int32_t* new_table, int32_t* new_refs, int32_t* page_map, int64_t entries,
                   int64_t pages, int64_t page, void* workspace, hipStream_t stream);
// paged_attn.hip
bool paged_attn_launchable(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                           int64_t max_blocks, int64_t page);
size_t paged_attn_workspace_bytes(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                                  int64_t max_blocks, int64_t page);
int paged_attn_run(const void* query, const void* query_rope, const void* key, const void* key_rope,
                   const void* value, void* out, float* smax, float* ssum, const int32_t* act_q,
                   const int32_t* act_k, const int32_t* table, int64_t batch, int64_t s1, int64_t n1, int64_t n2,
                   int64_t d, int64_t num_blocks, int64_t page, int64_t max_blocks, int32_t mode, int64_t pre_tokens,
                   int64_t next_tokens, int32_t dtype, float scale, int32_t return_lse, void* workspace,
                   hipStream_t stream);

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

static int check_caches(int64_t n, const void* const* caches, const int64_t* row_bytes, int64_t page) {
  DSA_CHECK_ARG(n >= 0 && n <= 65536, "number of caches must be in [0, 65536]");
  DSA_CHECK_ARG(n == 0 || (caches && row_bytes), "null cache list");
  for (int64_t i = 0; i < n; ++i) {
    DSA_CHECK_ARG(caches[i], "null cache pointer");
    DSA_CHECK_SUPPORTED(row_bytes[i] >= 1 && row_bytes[i] <= (1 << 24) && within(row_bytes[i], page, (1ll << 31) - 1),
                        "a cache row must have between 1 byte and 16 MiB, a page less than 2 GiB");
  }
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

}  // namespace dsa

using namespace dsa;

extern "C" {

int dsa_rope(const void* query, void* query_out, int64_t q_in_sb, int64_t q_in_ss, int64_t q_in_sh, int64_t q_out_sb,
             int64_t q_out_ss, int64_t q_out_sh, int64_t q_heads, int64_t q_d, int64_t q_start, const void* key,
             void* key_out, int64_t k_in_sb, int64_t k_in_ss, int64_t k_in_sh, int64_t k_out_sb, int64_t k_out_ss,
             int64_t k_out_sh, int64_t k_heads, int64_t k_d, int64_t k_start, const void* positions,
             int32_t positions_64, int32_t positions_per_sequence, const double* inv_freq, int64_t batch, int64_t s1,
             int64_t rotary_dim, int32_t interleaved, int32_t inverse, int32_t dtype, float attention_scale,
             void* stream) {
  clear_error();
  DSA_CHECK_ARG(query && query_out && positions && inv_freq, "null tensor pointer");
  DSA_CHECK_ARG((key == nullptr) == (key_out == nullptr), "key and key_out must be both provided or both omitted");
  DSA_CHECK_SUPPORTED(dtype == DSA_DTYPE_BF16 || dtype == DSA_DTYPE_FP16 || dtype == DSA_DTYPE_FP32,
                      "dtype must be bfloat16, float16 or float32");
  DSA_CHECK_SUPPORTED(rotary_dim >= 2 && rotary_dim <= 1024 && rotary_dim % 2 == 0,
                      "rotary dim must be even and in [2, 1024], got %lld", (long long)rotary_dim);
  DSA_CHECK_ARG(batch >= 1 && s1 >= 1 && batch < (1ll << 31) && s1 < (1ll << 31) && within(batch, s1, 1ll << 40),
                "batch and tokens must be in [1, 2^31)");
  const void* in[2] = {query, key};
  void* out[2] = {query_out, key_out};
  const int64_t heads[2] = {q_heads, k_heads}, d[2] = {q_d, k_d}, start[2] = {q_start, k_start};
  const int64_t qs[6] = {q_in_sb, q_in_ss, q_in_sh, q_out_sb, q_out_ss, q_out_sh};
  const int64_t ks[6] = {k_in_sb, k_in_ss, k_in_sh, k_out_sb, k_out_ss, k_out_sh};
  const int64_t* strides[2] = {qs, ks};
  const int n = key ? 2 : 1;
  for (int i = 0; i < n; ++i) {
    DSA_CHECK_ARG(heads[i] >= 1 && d[i] >= 1 && d[i] <= (1 << 20) && within(heads[i], d[i], 1 << 24),
                  "heads and head dim must be positive, heads * head dim at most 2^24");
    DSA_CHECK_ARG(start[i] >= 0 && start[i] <= d[i] - rotary_dim,
                  "the rotary slice [%lld, +%lld) must lie inside the head dim %lld", (long long)start[i],
                  (long long)rotary_dim, (long long)d[i]);
    for (int j = 0; j < 6; ++j)
      DSA_CHECK_ARG(strides[i][j] >= 0 && strides[i][j] < (1ll << 48), "strides must be in [0, 2^48)");
  }
  return rope_run(in, out, strides, heads, d, start, n, positions, positions_64, positions_per_sequence, inv_freq,
                  batch * s1, s1, rotary_dim, interleaved != 0, inverse != 0, dtype, attention_scale,
                  (hipStream_t)stream);
}

int dsa_paged_cache_write(int64_t n_caches, const void* const* rows, void* const* caches, const int64_t* row_bytes,
                          const int64_t* row_batch_stride, const int64_t* row_token_stride, const int32_t* block_table,
                          const int32_t* seq_lengths, const int32_t* row_lengths, int64_t batch, int64_t s1,
                          int64_t tokens, int64_t max_blocks, int64_t num_pages, int64_t page_size, int32_t layout,
                          void* stream) {
  clear_error();
  DSA_CHECK_ARG(n_caches >= 1 && rows && row_batch_stride && row_token_stride, "null row list");
  DSA_CHECK_ARG(block_table && seq_lengths, "null tensor pointer");
  int st = check_pages(num_pages, page_size, max_blocks);
  if (st != DSA_OK) return st;
  st = check_caches(n_caches, (const void* const*)caches, row_bytes, page_size);
  if (st != DSA_OK) return st;
  for (int64_t i = 0; i < n_caches; ++i) {
    DSA_CHECK_ARG(rows[i], "null row pointer");
    DSA_CHECK_ARG(row_batch_stride[i] >= 0 && row_token_stride[i] >= 0 && row_batch_stride[i] < (1ll << 48) &&
                      row_token_stride[i] < (1ll << 48),
                  "row strides must be in [0, 2^48)");
  }
  DSA_CHECK_SUPPORTED(layout == DSA_LAYOUT_BSND || layout == DSA_LAYOUT_TND, "layout must be BSND or TND");
  DSA_CHECK_ARG(batch >= 1 && batch <= (1 << 24), "batch must be in [1, 2^24]");
  DSA_CHECK_ARG(tokens >= 1 && tokens < (1ll << 31), "tokens must be in [1, 2^31)");
  if (layout == DSA_LAYOUT_TND)
    DSA_CHECK_ARG(row_lengths, "TND layout requires row_lengths (cumulative)");
  else
    DSA_CHECK_ARG(s1 >= 1 && s1 < (1ll << 31) && within(batch, s1, (1ll << 31) - 1) && batch * s1 == tokens,
                  "tokens must equal B*S for BSND rows");
  return pc_write_run(n_caches, rows, caches, row_bytes, row_batch_stride, row_token_stride, block_table, seq_lengths,
                      row_lengths, batch, s1, tokens, max_blocks, num_pages, page_size, layout, (hipStream_t)stream);
}

size_t dsa_paged_cache_fork_workspace_size(int64_t rows, int64_t new_rows, int64_t num_pages) {
  if (rows < 1 || rows > (1 << 24) || new_rows < 1 || new_rows > (1 << 24) || num_pages < 1 ||
      num_pages >= (1ll << 31))
    return 0;
  return pc_fork_workspace_bytes(rows, new_rows, num_pages);
}

int dsa_paged_cache_fork(int64_t n_caches, void* const* caches, const int64_t* row_bytes, const int32_t* block_table,
                         const int32_t* seq_lengths, const int32_t* page_refs, const int32_t* parents,
                         int32_t* new_block_table, int32_t* new_seq_lengths, int32_t* new_page_refs, int64_t rows,
                         int64_t new_rows, int64_t max_blocks, int64_t new_max_blocks, int64_t num_pages,
                         int64_t page_size, int64_t new_tokens, void* workspace, size_t workspace_bytes,
                         void* stream) {
  clear_error();
  DSA_CHECK_ARG(block_table && seq_lengths && page_refs && new_block_table && new_seq_lengths && new_page_refs,
                "null tensor pointer");
  int st = check_pages(num_pages, page_size, max_blocks);
  if (st != DSA_OK) return st;
  st = check_pages(num_pages, page_size, new_max_blocks);
  if (st != DSA_OK) return st;
  st = check_caches(n_caches, (const void* const*)caches, row_bytes, page_size);
  if (st != DSA_OK) return st;
  DSA_CHECK_ARG(rows >= 1 && rows <= (1 << 24) && new_rows >= 1 && new_rows <= (1 << 24),
                "rows of the block tables must be in [1, 2^24]");
  DSA_CHECK_ARG(parents || rows == new_rows, "without parents the new table has as many rows as the old");
  DSA_CHECK_ARG(new_tokens >= 0 && new_tokens < (1ll << 31), "new_tokens must be in [0, 2^31)");
  DSA_CHECK_ARG(block_table != new_block_table && seq_lengths != new_seq_lengths && page_refs != new_page_refs,
                "the new tables must not be the old ones");
  st = check_workspace(workspace, workspace_bytes, pc_fork_workspace_bytes(rows, new_rows, num_pages));
  if (st != DSA_OK) return st;
  return pc_fork_run(n_caches, caches, row_bytes, block_table, seq_lengths, page_refs, parents, new_block_table,
                     new_seq_lengths, new_page_refs, rows, new_rows, max_blocks, new_max_blocks, num_pages, page_size,
                     new_tokens, workspace, (hipStream_t)stream);
}

size_t dsa_paged_cache_compact_workspace_size(int64_t num_pages) {
  if (num_pages < 1 || num_pages >= (1ll << 31)) return 0;
  return pc_compact_workspace_bytes(num_pages);
}

int dsa_paged_cache_compact(int64_t n_caches, void* const* caches, const int64_t* row_bytes,
                            const int32_t* block_table, const int32_t* page_refs, int32_t* new_block_table,
                            int32_t* new_page_refs, int32_t* page_map, int64_t rows, int64_t max_blocks,
                            int64_t num_pages, int64_t page_size, void* workspace, size_t workspace_bytes,
                            void* stream) {
  clear_error();
  DSA_CHECK_ARG(block_table && page_refs && new_block_table && new_page_refs && page_map, "null tensor pointer");
  int st = check_pages(num_pages, page_size, max_blocks);
  if (st != DSA_OK) return st;
  st = check_caches(n_caches, (const void* const*)caches, row_bytes, page_size);
  if (st != DSA_OK) return st;
  DSA_CHECK_ARG(rows >= 1 && rows <= (1 << 24), "rows of the block table must be in [1, 2^24]");
  DSA_CHECK_ARG(page_refs != new_page_refs && page_refs != page_map && new_page_refs != page_map,
                "the new counts and the page map must be arrays of their own");
  st = check_workspace(workspace, workspace_bytes, pc_compact_workspace_bytes(num_pages));
  if (st != DSA_OK) return st;
  return pc_compact_run(n_caches, caches, row_bytes, block_table, page_refs, new_block_table, new_page_refs, page_map,
                        rows * max_blocks, num_pages, page_size, workspace, (hipStream_t)stream);
}

size_t dsa_paged_attn_workspace_size(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, int32_t latent,
                                     int64_t max_blocks, int64_t page_size) {
  if (!paged_attn_sizes_ok(batch, s1, n1, n2, d, latent != 0, max_blocks, page_size)) return 0;
  return paged_attn_workspace_bytes(batch, s1, n1, n2, d, latent != 0, max_blocks, page_size);
}

int dsa_paged_attn(const void* query, const void* query_rope, const void* key, const void* key_rope,
                   const void* value, void* attention_out, float* softmax_max, float* softmax_sum,
                   const int32_t* actual_seq_q, const int32_t* actual_seq_kv, const int32_t* block_table,
                   int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, int64_t d_rope, int64_t num_blocks,
                   int64_t page_size, int64_t max_blocks, int32_t sparse_mode, int64_t pre_tokens,
                   int64_t next_tokens, int32_t dtype, float scale_value, int32_t return_lse, void* workspace,
                   size_t workspace_bytes, void* stream) {
  clear_error();
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
  st = check_workspace(workspace, workspace_bytes,
                       paged_attn_workspace_bytes(batch, s1, n1, n2, d, latent, max_blocks, page_size));
  if (st != DSA_OK) return st;
  DSA_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "the workspace must be 16-byte aligned");
  return paged_attn_run(query, query_rope, key, key_rope, value, attention_out, softmax_max, softmax_sum, actual_seq_q,
                        actual_seq_kv, block_table, batch, s1, n1, n2, d, num_blocks, page_size, max_blocks,
                        sparse_mode, pre_tokens, next_tokens, dtype, scale_value, return_lse, workspace,
                        (hipStream_t)stream);
}

}  // extern "C"
