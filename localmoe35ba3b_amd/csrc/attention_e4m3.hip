// Attention over a paged cache of 8-bit values with scales (attention.hpp has the kernels).
#include "attention.hpp"

using namespace lm;

extern "C" int lm_paged_attention_e4m3(
    const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads,
    const void *k_pages, const void *v_pages, const float *scales, int64_t scale_stride,
    int64_t pages, int64_t page_stride, int64_t kv_heads, int64_t page_size, int64_t head_dim,
    const int32_t *starts, const int32_t *lengths, const int32_t *table, int64_t table_stride,
    int64_t table_pages, int64_t sequences, int64_t tokens, int64_t max_new, float scale,
    const void *gate, int64_t gate_token_stride, int64_t gate_head_stride, void *out,
    void *workspace, int64_t workspace_bytes, int dtype, void *stream) {
  return paged_attention<true>(
      q, q_token_stride, q_head_stride, q_heads, k_pages, v_pages, scales, scale_stride, pages,
      page_stride, kv_heads, page_size, head_dim, starts, lengths, table, table_stride, table_pages,
      sequences, tokens, max_new, scale, gate, gate_token_stride, gate_head_stride, out, workspace,
      workspace_bytes, dtype, stream);
}
