// Attention of each sequence's new tokens over its paged cache (gfx950).
//
//   o_t = sum_{j <= p_t} e^{scale q_t.k_j - m_t} v_j / sum_j e^{scale q_t.k_j - m_t}
//
// causal at the end of the sequence, times sigmoid(gate_t) where a gate is given;
// a row without a visible key is 0.
//
// One wave takes one (token, query head) and walks its keys 64 at a time: lane j
// forms key j's score, then the wave adds the weighted values, each lane its
// D / 64 channels.
#include "paged.hpp"

namespace lm {
namespace {

struct Attention {
  const uint16_t *q, *gate;  // gate: null or a row for each row of q
  int64_t q_token, q_head, gate_token, gate_head;  // strides, elements
  const uint16_t *k_pages, *v_pages;
  uint16_t *out;  // [tokens][q_heads][D]
  PagedBatch batch;
  int tokens, q_heads, group;
  float scale;
};

template <typename T, int D>
__global__ __launch_bounds__(64) void attention_row_kernel(Attention a) {
  const int t = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  const int s = paged_find(a.batch, t);
  if (s < 0) return;  // a row of no sequence keeps its output
  const PagedSequence seq = paged_sequence(a.batch, s, a.tokens);
  const int keys = min(seq.base + (t - seq.first) + 1, seq.length);
  const int kv = head / a.group, shift = a.batch.page_shift, mask = (1 << shift) - 1;
  constexpr int C = D / 64;
  __shared__ float qs[D], ps[64];
  for (int i = lane; i < D; i += 64)
    qs[i] = T::to_f32(a.q[t * a.q_token + head * a.q_head + i]) * a.scale;
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o[C] = {};
  for (int k0 = 0; k0 < keys; k0 += 64) {
    const int j = k0 + lane;
    float x = -INFINITY;
    if (j < keys) {
      const uint16_t *kr =
          a.k_pages + paged_page(a.batch, s, j) + ((int64_t)(kv << shift) + (j & mask)) * D;
      x = 0.0f;
      for (int i = 0; i < D; ++i) x = __builtin_fmaf(qs[i], T::to_f32(kr[i]), x);
    }
    float mx = x;
    for (int i = 32; i >= 1; i >>= 1) mx = fmaxf(mx, __shfl_xor(mx, i, 64));
    const float mn = fmaxf(m, mx), at = mn == -INFINITY ? 0.0f : mn;
    const float keep = expf(m - at), p = expf(x - at);
    m = mn;
    l = l * keep + wave_sum_f32(p);
    ps[lane] = p;
    __syncthreads();
    for (int c = 0; c < C; ++c) o[c] *= keep;
    for (int i = 0; i < min(64, keys - k0); ++i) {
      const uint16_t *vr = a.v_pages + paged_page(a.batch, s, k0 + i) +
                           ((int64_t)(kv << shift) + ((k0 + i) & mask)) * D;
      for (int c = 0; c < C; ++c)
        o[c] = __builtin_fmaf(ps[i], T::to_f32(vr[c * 64 + lane]), o[c]);
    }
    __syncthreads();
  }
  for (int c = 0; c < C; ++c) {
    const int i = c * 64 + lane;
    float y = keys > 0 ? o[c] / l : 0.0f;
    if (a.gate) y *= sigmoid_f32(T::to_f32(a.gate[t * a.gate_token + head * a.gate_head + i]));
    a.out[((int64_t)t * a.q_heads + head) * D + i] = T::from_f32(y);
  }
}

template <typename T>
int launch_attention(const Attention &a, int head_dim, hipStream_t st) {
  const dim3 grid(a.tokens, a.q_heads);
  if (head_dim == 256)
    attention_row_kernel<T, 256><<<grid, 64, 0, st>>>(a);
  else if (head_dim == 128)
    attention_row_kernel<T, 128><<<grid, 64, 0, st>>>(a);
  else
    attention_row_kernel<T, 64><<<grid, 64, 0, st>>>(a);
  return check_launch("attention_row_kernel");
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int64_t lm_paged_attention_workspace_bytes(int64_t tokens, int64_t sequences,
                                                      int64_t q_heads, int64_t kv_heads,
                                                      int64_t head_dim, int64_t max_new) {
  return 0;
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
  if (const int rc = paged_check(pages, page_stride, kv_heads, page_size, head_dim, starts, lengths,
                                 table, table_stride, table_pages, sequences, tokens, dtype))
    return rc;
  LM_REQUIRE(q_heads >= 1 && q_heads <= 65536 && q_heads % kv_heads == 0, LM_EINVAL,
             "query heads must be a multiple of key-value heads");
  LM_REQUIRE(max_new >= 0, LM_EINVAL, "invalid number of new tokens");
  if (tokens == 0 || sequences == 0) return LM_OK;
  LM_REQUIRE(q && k_pages && v_pages && out, LM_EINVAL, "null pointer");
  LM_REQUIRE(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out) &&
                 q_token_stride % 8 == 0 && q_head_stride % 8 == 0 && q_token_stride >= 0 &&
                 q_head_stride >= 0,
             LM_EINVAL, "head rows must be 16-byte aligned");
  LM_REQUIRE(!gate || (aligned16(gate) && gate_token_stride % 8 == 0 && gate_head_stride % 8 == 0 &&
                       gate_token_stride >= 0 && gate_head_stride >= 0),
             LM_EINVAL, "head rows must be 16-byte aligned");
  Attention a = {};
  a.q = static_cast<const uint16_t *>(q), a.q_token = q_token_stride, a.q_head = q_head_stride;
  a.gate = static_cast<const uint16_t *>(gate);
  a.gate_token = gate_token_stride, a.gate_head = gate_head_stride;
  a.k_pages = static_cast<const uint16_t *>(k_pages);
  a.v_pages = static_cast<const uint16_t *>(v_pages);
  a.out = static_cast<uint16_t *>(out);
  a.batch = {starts, lengths, table, table_stride, (int)sequences, (int)table_pages,
             __builtin_ctzll((unsigned long long)page_size), (int)pages, page_stride,
             (int)kv_heads};
  a.tokens = (int)tokens, a.q_heads = (int)q_heads, a.group = (int)(q_heads / kv_heads);
  a.scale = scale;
  return dtype == LM_BF16 ? launch_attention<BF16>(a, (int)head_dim, as_stream(stream))
                          : launch_attention<FP16>(a, (int)head_dim, as_stream(stream));
}
