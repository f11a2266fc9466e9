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
// A workgroup takes the rows of a token; D / 8 lanes hold one.  A lane of the rotated
// channels takes four of the first half and their four partners of the second, others eight
// in a row, so the rotation needs no exchange and a row is read once.  The first rows are
// requested at the start, beside the position, whose lookups (sequence, length, page) are
// the longest chain of a small call.
//
// Bound by the rows' bytes where there are many, by that chain where there are few.  18 heads
// of 256: 4096 tokens 16 us (75.5 MB, 4.7 TB/s), one token 3 us; 64 tokens into a cache 5 us;
// 3310 tokens into a cache (48 heads of 128) 18 us (81 MB, 4.6 TB/s).
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
constexpr int kAhead = 3;  // rows of a thread that are requested together

// Sum over the LANES (8, 16 or 32) lanes of a row, in every lane.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (LANES == 8) return octet_sum_f32(v);
  v = row_sum_f32(v);
  if constexpr (LANES == 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

struct Row8 {
  uint2 lo, hi;
};

template <typename T>
__device__ __forceinline__ void unpack4(uint2 w, float x[4]) {
  x[0] = T::to_f32(w.x & 0xFFFFu), x[1] = T::to_f32(w.x >> 16);
  x[2] = T::to_f32(w.y & 0xFFFFu), x[3] = T::to_f32(w.y >> 16);
}

template <typename T, int LANES, bool PAGED>
__global__ __launch_bounds__(256) void head_rows_kernel(HeadRows a) {
  constexpr int D = LANES * 8, ROWS = 256 / LANES;
  __shared__ __attribute__((aligned(16))) float cosines[kMaxHalf], sines[kMaxHalf];
  __shared__ int64_t place;  // element offset of the token's row of head 0 in the cache; < 0: none
  __shared__ int found, at;  // the token's sequence and position
  const int t = blockIdx.x, tid = threadIdx.x, lane = tid % LANES, half = a.half;
  const int heads = a.q_heads + a.k_heads + (PAGED ? a.k_heads : 0);
  const bool rotated = lane * 8 < 2 * half;
  const int lo = rotated ? lane * 4 : lane * 8, hi = rotated ? half + lane * 4 : lane * 8 + 4;

  auto load = [&](int r) {  // row r of the token: its queries, then keys, then values
    r = min(r, heads - 1);
    const uint16_t *p = r < a.q_heads ? a.q + t * a.q_token + r * a.q_head
                        : r < a.q_heads + a.k_heads
                            ? a.k + t * a.k_token + (r - a.q_heads) * a.k_head
                            : a.v + t * a.v_token + (r - a.q_heads - a.k_heads) * a.v_head;
    return Row8{ldg_u2(p + lo), ldg_u2(p + hi)};
  };
  const int r0 = tid / LANES;
  Row8 raw[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) raw[i] = load(r0 + i * ROWS);
  const float freq = tid < half ? a.inv_freq[tid] : 0.0f;

  double position;
  int64_t to = 0;
  if constexpr (PAGED) {
    if (tid == 0) found = -1;
    __syncthreads();
    for (int s = tid; s < a.batch.sequences; s += 256) {
      const int first = a.batch.starts[s], end = a.batch.starts[s + 1], n = a.batch.lengths[s];
      if (first <= t && t < end) found = s, at = n - (end - first) + (t - first);
    }
    __syncthreads();
    if (found < 0) {  // a row of no sequence
      for (int r = r0; r < a.q_heads; r += ROWS) {
        uint16_t *dst = a.q_out + ((int64_t)t * a.q_heads + r) * D;
        *reinterpret_cast<uint2 *>(dst + lo) = *reinterpret_cast<uint2 *>(dst + hi) = uint2{0, 0};
      }
      return;
    }
    const int p = at;
    position = p;
    if (tid == 255) {
      const int64_t room = (int64_t)a.batch.table_pages << a.batch.page_shift;
      place = p < 0 || p >= room ? -1
                                 : paged_page(a.batch, found, p) +
                                       (int64_t)(p & ((1 << a.batch.page_shift) - 1)) * D;
    }
  } else {
    position = (double)a.positions[t];
  }
  if (tid < half) {
    constexpr double kTurns = 0.15915494309189533577;  // 1 / (2 pi)
    const double turns = position * (double)freq * kTurns;
    sincospif(2.0f * (float)(turns - rint(turns)), &sines[tid], &cosines[tid]);
  }
  __syncthreads();
  if constexpr (PAGED) to = place;

  float c[4], s[4];
  if (rotated) {
    *reinterpret_cast<float4 *>(c) = *reinterpret_cast<const float4 *>(cosines + lo);
    *reinterpret_cast<float4 *>(s) = *reinterpret_cast<const float4 *>(sines + lo);
  }
  for (int r = r0; r < heads;) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i, r += ROWS) {
      if (r >= heads) break;
      float x[4], y[4];
      unpack4<T>(raw[i].lo, x);
      unpack4<T>(raw[i].hi, y);
      const bool value = PAGED && r >= a.q_heads + a.k_heads;
      const float *w = r < a.q_heads ? a.q_w : value ? nullptr : a.k_w;
      if (w) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(x[j], x[j], ss);
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(y[j], y[j], ss);
        const float n = 1.0f / sqrtf(lanes_sum<LANES>(ss) * (1.0f / D) + a.eps);
        const float4 w0 = *reinterpret_cast<const float4 *>(w + lo);
        const float4 w1 = *reinterpret_cast<const float4 *>(w + hi);
        x[0] *= n * (1.0f + w0.x), x[1] *= n * (1.0f + w0.y);
        x[2] *= n * (1.0f + w0.z), x[3] *= n * (1.0f + w0.w);
        y[0] *= n * (1.0f + w1.x), y[1] *= n * (1.0f + w1.y);
        y[2] *= n * (1.0f + w1.z), y[3] *= n * (1.0f + w1.w);
      }
      if (rotated && !value) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float u = x[j] * c[j] - y[j] * s[j];
          y[j] = y[j] * c[j] + x[j] * s[j];
          x[j] = u;
        }
      }
      uint16_t *dst;
      if (r < a.q_heads) {
        dst = a.q_out + ((int64_t)t * a.q_heads + r) * D;
      } else {
        const int h = r - a.q_heads - (value ? a.k_heads : 0);
        if constexpr (PAGED) {
          if (to < 0) continue;
          dst = (value ? a.v_pages : a.k_pages) + to + ((int64_t)h << a.batch.page_shift) * D;
        } else {
          dst = a.k_out + ((int64_t)t * a.k_heads + h) * D;
        }
      }
      *reinterpret_cast<uint2 *>(dst + lo) = uint2{T::pack2(x[0], x[1]), T::pack2(x[2], x[3])};
      *reinterpret_cast<uint2 *>(dst + hi) = uint2{T::pack2(y[0], y[1]), T::pack2(y[2], y[3])};
    }
    if (r < heads) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) raw[i] = load(r + i * ROWS);
    }
  }
}

template <typename T, bool PAGED>
void launch_rows(const HeadRows &a, int head_dim, hipStream_t st) {
  const unsigned grid = (unsigned)a.tokens;
  if (head_dim == 256)
    head_rows_kernel<T, 32, PAGED><<<grid, 256, 0, st>>>(a);
  else if (head_dim == 128)
    head_rows_kernel<T, 16, PAGED><<<grid, 256, 0, st>>>(a);
  else
    head_rows_kernel<T, 8, PAGED><<<grid, 256, 0, st>>>(a);
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
  LM_REQUIRE(tokens >= 0 && tokens < kMaxTokens, LM_EINVAL, "invalid token count");
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
