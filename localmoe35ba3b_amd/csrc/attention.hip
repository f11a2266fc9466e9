// Attention over a paged cache of the rows' own type (attention.hpp has the kernels).
#include "attention.hpp"

using namespace lm;

extern "C" int64_t lm_paged_attention_workspace_bytes(int64_t tokens, int64_t sequences,
                                                      int64_t q_heads, int64_t kv_heads,
                                                      int64_t head_dim, int64_t max_new,
                                                      int64_t max_keys) {
  if (tokens < 1 || sequences < 1 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads ||
      max_new < 0)
    return 0;
  return attention_bytes(
      attention_plan(tokens, sequences, q_heads, kv_heads, head_dim, max_new, max_keys), head_dim);
}

extern "C" int lm_paged_attention(const void *q, int64_t q_token_stride, int64_t q_head_stride,
                                  int64_t q_heads, const void *k_pages, const void *v_pages,
                                  int64_t pages, int64_t page_stride, int64_t kv_heads,
                                  int64_t page_size, int64_t head_dim, const int32_t *starts,
                                  const int32_t *lengths, const int32_t *table,
                                  int64_t table_stride, int64_t table_pages, int64_t sequences,
                                  int64_t tokens, int64_t max_new, float scale, const void *gate,
                                  int64_t gate_token_stride, int64_t gate_head_stride, void *out,
                                  void *workspace, int64_t workspace_bytes, int dtype,
                                  void *stream) {
  return paged_attention<false>(
      q, q_token_stride, q_head_stride, q_heads, k_pages, v_pages, nullptr, 0, pages, page_stride,
      kv_heads, page_size, head_dim, starts, lengths, table, table_stride, table_pages, sequences,
      tokens, max_new, scale, gate, gate_token_stride, gate_head_stride, out, workspace,
      workspace_bytes, dtype, stream);
}
