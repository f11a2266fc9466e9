// Per-head rows on their way into attention (gfx950): norms of queries and keys,
// the position rotation, and the append of keys and values to a paged cache.
//
//   n = x * rsqrt(mean_d x^2 + eps) * (1 + w)                    (no w: n = x)
//   y_i = n_i cos a_i - n_{i+h} sin a_i,  y_{i+h} = n_{i+h} cos a_i + n_i sin a_i
//   a_i = position * inv_freq_i,  i < h;  channels from 2 h on: y = n
//
// in fp32, rounded once.  Positions reach hundreds of thousands, where an fp32
// angle is off by a hundredth of a turn: the product of a position and an fp32
// frequency is exact in fp64, and its turns are reduced there before sine and
// cosine are taken in fp32.
//
// A workgroup takes the rows of a few tokens.  Its threads first form each
// token's angles once, in LDS; then D / 8 lanes hold a row, 16 bytes each, so a
// row is read once, its sum of squares is a lane reduction, and the rotation's
// partner channel is a lane shuffle.
#include "paged.hpp"

namespace lm {
namespace {

struct HeadRows {
  const uint16_t *q, *k, *v;  // null: not in this call
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides, elements
  uint16_t *q_out, *k_out;    // [tokens][heads][D]; k_out only without a cache
  uint16_t *k_pages, *v_pages;
  const float *q_w, *k_w, *inv_freq;  // null: no norm, no rotation
  const int64_t *positions;           // without a cache
  PagedBatch batch;
  int tokens, q_heads, k_heads;
  int half;  // rotated pairs
  float eps;
};

constexpr int kMaxHalf = 128;

// LANES = D / 8 lanes hold a row.  TOKENS per workgroup.
template <typename T, int LANES, int TOKENS, bool PAGED>
__global__ __launch_bounds__(256) void head_rows_kernel(HeadRows a) {
  constexpr int D = LANES * 8, ROWS = 256 / LANES;
  __shared__ float cosines[TOKENS][kMaxHalf], sines[TOKENS][kMaxHalf];
  __shared__ int64_t place[TOKENS];     // element offset of the token's row of head 0; < 0: none
  __shared__ double position[TOKENS];
  const int t0 = blockIdx.x * TOKENS, n = min(TOKENS, a.tokens - t0);
  if (threadIdx.x < n) {
    const int t = t0 + threadIdx.x;
    if constexpr (PAGED) {
      const int s = paged_find(a.batch, t);
      int64_t at = -1;
      int p = 0;
      if (s >= 0) {
        const int first = a.batch.starts[s], count = a.batch.starts[s + 1] - first;
        p = a.batch.lengths[s] - count + (t - first);
        const int64_t room = (int64_t)a.batch.table_pages << a.batch.page_shift;
        at = -2;  // a token of the sequence without a place in the cache
        if (p >= 0 && p < room)
          at = paged_page(a.batch, s, p) + (int64_t)(p & ((1 << a.batch.page_shift) - 1)) * D;
      }
      place[threadIdx.x] = at;
      position[threadIdx.x] = p;
    } else {
      place[threadIdx.x] = 0;
      position[threadIdx.x] = (double)a.positions[t];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * a.half; i += 256) {
    const int t = i / a.half, j = i - t * a.half;
    constexpr double kTurns = 0.15915494309189533577;  // 1 / (2 pi)
    const double turns = position[t] * (double)a.inv_freq[j] * kTurns;
    const float r = (float)(turns - rint(turns));
    sincospif(2.0f * r, &sines[t][j], &cosines[t][j]);
  }
  __syncthreads();

  const int lane = threadIdx.x % LANES, e0 = lane * 8, half = a.half;
  const int heads = a.q_heads + a.k_heads + (PAGED ? a.k_heads : 0);
  const bool rotated = e0 < 2 * half;
  const int partner = (threadIdx.x & 63) + (rotated ? (e0 < half ? half / 8 : -half / 8) : 0);
  for (int r = threadIdx.x / LANES; r < n * heads; r += ROWS) {
    const int tl = r / heads, t = t0 + tl;
    int h = r - tl * heads;
    const int64_t at = place[tl];
    const uint16_t *src;
    uint16_t *dst;
    const float *w = nullptr;
    bool turn = half > 0;
    if (h < a.q_heads) {
      src = a.q + t * a.q_token + h * a.q_head;
      dst = a.q_out + ((int64_t)t * a.q_heads + h) * D;
      if (at == -1) continue;  // a row of no sequence
      w = a.q_w;
    } else {
      h -= a.q_heads;
      const int64_t to = at + ((int64_t)h << a.batch.page_shift) * D;
      if (h < a.k_heads) {
        src = a.k + t * a.k_token + h * a.k_head;
        dst = PAGED ? a.k_pages + to : a.k_out + ((int64_t)t * a.k_heads + h) * D;
        w = a.k_w;
      } else {
        h -= a.k_heads;
        src = a.v + t * a.v_token + h * a.v_head;
        dst = a.v_pages + (to - ((int64_t)a.k_heads << a.batch.page_shift) * D);
        turn = false;
      }
      if (at < 0) continue;
    }
    const u32x4 raw = ldg16(src + e0);
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = T::to_f32(raw[i] & 0xFFFFu);
      x[2 * i + 1] = T::to_f32(raw[i] >> 16);
    }
    if (w) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
#pragma unroll
      for (int o = LANES / 2; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, 64);
      const float s = 1.0f / sqrtf(ss * (1.0f / D) + a.eps);
      const float4 w0 = *reinterpret_cast<const float4 *>(w + e0);
      const float4 w1 = *reinterpret_cast<const float4 *>(w + e0 + 4);
      const float wv[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * s * (1.0f + wv[i]);
    }
    if (turn) {
      const int j = rotated ? (e0 < half ? e0 : e0 - half) : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float other = __shfl(x[i], partner, 64);
        const float c = cosines[tl][j + i], s = sines[tl][j + i];
        if (rotated) x[i] = x[i] * c + (e0 < half ? -other * s : other * s);
      }
    }
    u32x4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = T::pack2(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<u32x4 *>(dst + e0) = y;
  }
}

template <typename T, bool PAGED>
void launch_rows(const HeadRows &a, int head_dim, hipStream_t st) {
  constexpr int TOKENS = 4;
  const unsigned grid = cdiv(a.tokens, TOKENS);
  if (head_dim == 256)
    head_rows_kernel<T, 32, TOKENS, PAGED><<<grid, 256, 0, st>>>(a);
  else if (head_dim == 128)
    head_rows_kernel<T, 16, TOKENS, PAGED><<<grid, 256, 0, st>>>(a);
  else
    head_rows_kernel<T, 8, TOKENS, PAGED><<<grid, 256, 0, st>>>(a);
}

// Checks of one input's rows, whose head_dim channels are contiguous.
int check_rows(const void *p, int64_t token, int64_t head, const float *w) {
  LM_REQUIRE(p && aligned16(p) && token % 8 == 0 && head % 8 == 0 && token >= 0 && head >= 0,
             LM_EINVAL, "head rows must be 16-byte aligned");
  LM_REQUIRE(!w || aligned16(w), LM_EINVAL, "norm weights must be 16-byte aligned");
  return LM_OK;
}

int check_rotation(const float *inv_freq, int64_t pairs, int64_t head_dim) {
  if (!inv_freq) {
    LM_REQUIRE(pairs == 0, LM_EINVAL, "null pointer");
    return LM_OK;
  }
  LM_REQUIRE(pairs >= 8 && pairs % 8 == 0 && 2 * pairs <= head_dim, LM_EINVAL,
             "rotated channels must be a multiple of 16 and fit the head");
  return LM_OK;
}

}  // namespace
}  // namespace lm

using namespace lm;

extern "C" int lm_qk_norm_rope(const void *q, int64_t q_token_stride, int64_t q_head_stride,
                               int64_t q_heads, const float *q_weight, void *q_out, const void *k,
                               int64_t k_token_stride, int64_t k_head_stride, int64_t k_heads,
                               const float *k_weight, void *k_out, const int64_t *positions,
                               const float *inv_freq, int64_t pairs, int64_t tokens,
                               int64_t head_dim, float eps, int dtype, void *stream) {
  LM_REQUIRE(dtype == LM_BF16 || dtype == LM_FP16, LM_EINVAL, "attention requires FP16/BF16");
  LM_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, LM_EINVAL,
             "attention supports heads of 64, 128 or 256");
  LM_REQUIRE(q_heads >= 0 && q_heads <= 65536 && k_heads >= 0 && k_heads <= 65536, LM_EINVAL,
             "invalid number of heads");
  LM_REQUIRE(tokens >= 0 && tokens < (1LL << 31), LM_EINVAL, "invalid token count");
  if (const int rc = check_rotation(inv_freq, pairs, head_dim)) return rc;
  if (tokens == 0 || q_heads + k_heads == 0) return LM_OK;
  if (q_heads)
    if (const int rc = check_rows(q, q_token_stride, q_head_stride, q_weight)) return rc;
  if (k_heads)
    if (const int rc = check_rows(k, k_token_stride, k_head_stride, k_weight)) return rc;
  LM_REQUIRE((!q_heads || (q_out && aligned16(q_out))) && (!k_heads || (k_out && aligned16(k_out))),
             LM_EINVAL, "head rows must be 16-byte aligned");
  LM_REQUIRE(positions, LM_EINVAL, "null pointer");
  HeadRows a = {};
  a.q = static_cast<const uint16_t *>(q);
  a.q_token = q_token_stride, a.q_head = q_head_stride, a.q_heads = (int)q_heads;
  a.q_w = q_weight, a.q_out = static_cast<uint16_t *>(q_out);
  a.k = static_cast<const uint16_t *>(k);
  a.k_token = k_token_stride, a.k_head = k_head_stride, a.k_heads = (int)k_heads;
  a.k_w = k_weight, a.k_out = static_cast<uint16_t *>(k_out);
  a.positions = positions, a.inv_freq = inv_freq, a.half = (int)pairs;
  a.tokens = (int)tokens, a.eps = eps;
  if (dtype == LM_BF16)
    launch_rows<BF16, false>(a, (int)head_dim, as_stream(stream));
  else
    launch_rows<FP16, false>(a, (int)head_dim, as_stream(stream));
  return check_launch("head_rows_kernel");
}

extern "C" int lm_paged_append(const void *k, int64_t k_token_stride, int64_t k_head_stride,
                               const float *k_weight, const void *v, int64_t v_token_stride,
                               int64_t v_head_stride, const void *q, int64_t q_token_stride,
                               int64_t q_head_stride, int64_t q_heads, const float *q_weight,
                               void *q_out, void *k_pages, void *v_pages, int64_t pages,
                               int64_t page_stride, int64_t kv_heads, int64_t page_size,
                               int64_t head_dim, const int32_t *starts, const int32_t *lengths,
                               const int32_t *table, int64_t table_stride, int64_t table_pages,
                               int64_t sequences, const float *inv_freq, int64_t pairs,
                               int64_t tokens, float eps, int dtype, void *stream) {
  if (const int rc = paged_check(pages, page_stride, kv_heads, page_size, head_dim, starts, lengths,
                                 table, table_stride, table_pages, sequences, tokens, dtype))
    return rc;
  LM_REQUIRE(q_heads >= 0 && q_heads <= 65536, LM_EINVAL, "invalid number of heads");
  if (const int rc = check_rotation(inv_freq, pairs, head_dim)) return rc;
  if (tokens == 0 || sequences == 0) return LM_OK;
  if (const int rc = check_rows(k, k_token_stride, k_head_stride, k_weight)) return rc;
  if (const int rc = check_rows(v, v_token_stride, v_head_stride, nullptr)) return rc;
  if (q_heads) {
    if (const int rc = check_rows(q, q_token_stride, q_head_stride, q_weight)) return rc;
    LM_REQUIRE(q_out && aligned16(q_out), LM_EINVAL, "head rows must be 16-byte aligned");
  }
  LM_REQUIRE(k_pages && v_pages && aligned16(k_pages) && aligned16(v_pages), LM_EINVAL,
             "pages must be 16-byte aligned");
  HeadRows a = {};
  a.k = static_cast<const uint16_t *>(k), a.v = static_cast<const uint16_t *>(v);
  a.k_token = k_token_stride, a.k_head = k_head_stride, a.k_heads = (int)kv_heads;
  a.v_token = v_token_stride, a.v_head = v_head_stride, a.k_w = k_weight;
  a.q = static_cast<const uint16_t *>(q);
  a.q_token = q_token_stride, a.q_head = q_head_stride, a.q_heads = (int)q_heads;
  a.q_w = q_weight, a.q_out = static_cast<uint16_t *>(q_out);
  a.k_pages = static_cast<uint16_t *>(k_pages), a.v_pages = static_cast<uint16_t *>(v_pages);
  a.batch = {starts, lengths, table, table_stride, (int)sequences, (int)table_pages,
             __builtin_ctzll((unsigned long long)page_size), (int)pages, page_stride,
             (int)kv_heads};
  a.inv_freq = inv_freq, a.half = (int)pairs, a.tokens = (int)tokens, a.eps = eps;
  if (dtype == LM_BF16)
    launch_rows<BF16, true>(a, (int)head_dim, as_stream(stream));
  else
    launch_rows<FP16, true>(a, (int)head_dim, as_stream(stream));
  return check_launch("head_rows_kernel");
}
