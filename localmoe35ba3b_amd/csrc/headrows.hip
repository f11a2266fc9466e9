// Per-head rows on their way into attention (gfx950): norms of queries and keys,
// the position rotation, and the append of keys and values to a paged cache.
//
//   n = x * rsqrt(mean_d x^2 + eps) * (1 + w)                    (no w: n = x)
//   y_i = n_i cos a_i - n_{i+h} sin a_i,  y_{i+h} = n_{i+h} cos a_i + n_i sin a_i
//   a_i = position * inv_freq_i,  i < h;  channels from 2 h on: y = n
//
// where a pair's position is that of its axis, if positions have several (time, row, column).
// In fp32, rounded once.  Positions reach hundreds of thousands, where an fp32
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
// Bound by the rows' bytes where there are many, by that chain where there are few.  From memory,
// 18 heads of 256: 4096 tokens 18 us (75.5 MB, 4.2 TB/s; 16.5 us with the rows in the caches), one
// token 3 us, of three axes too; 64 tokens into a cache 4 us; 3310 tokens into a cache (48 heads of
// 128) 21.5 us (81 MB, 3.8 TB/s; 18.4).
#include "paged.hpp"

namespace lm {
namespace {

struct HeadRows {
  const uint16_t *q, *k, *v;  // null: not in this call
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides, elements
  uint16_t *q_out, *k_out;    // [tokens][heads][D]; k_out only without a cache
  uint16_t *k_pages, *v_pages;
  const float *q_w, *k_w, *inv_freq;  // null: no norm, no rotation
  const int64_t *positions;           // [axes][tokens]; null: by the place in the sequence
  int64_t position_stride;            // between axes
  const int32_t *axis;                // of each pair; null: the first
  int axes;
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

// Sine and cosine of pair i of token t, at position p unless the call gives positions.
__device__ __forceinline__ void turn(const HeadRows &a, float freq, int i, int t, int p, float *s,
                                     float *c) {
  double position = p;
  if (a.positions) {
    const int axis = a.axis ? clamp_index32(a.axis[i], a.axes) : 0;
    position = (double)a.positions[axis * a.position_stride + t];
  }
  constexpr double kTurns = 0.15915494309189533577;  // 1 / (2 pi)
  const double turns = position * (double)freq * kTurns;
  sincospif(2.0f * (float)(turns - rint(turns)), s, c);
}

// The sequence of row t, negative for none, and its position there.  All 256 threads; of up to 64
// sequences each wave looks by itself.
struct TokenPlace {
  int s, position;
};
__device__ __forceinline__ TokenPlace find_token(const HeadRows &a, int t) {
  __shared__ int found, at;
  const int tid = threadIdx.x, S = a.batch.sequences;
  if (S <= 64) {
    const int k = min(tid & 63, S - 1);
    int first = a.batch.starts[k], end = a.batch.starts[k + 1], n = a.batch.lengths[k];
    asm volatile("" : "+v"(first), "+v"(end), "+v"(n));  // looked up together
    const uint64_t hit = __ballot(first <= t && t < end);
    if (!hit) return {-1, 0};
    const int s = min((int)__builtin_ctzll(hit), S - 1);
    return {s, __builtin_amdgcn_readlane(n - (end - first) + (t - first), s)};
  }
  if (tid == 0) found = -1;
  __syncthreads();
  for (int s = tid; s < S; s += 256) {
    const int first = a.batch.starts[s], end = a.batch.starts[s + 1], n = a.batch.lengths[s];
    if (first <= t && t < end) found = s, at = n - (end - first) + (t - first);
  }
  __syncthreads();
  return {found, at};
}

// The rows of token t.
template <typename T, int LANES, bool PAGED>
__device__ __forceinline__ void token_rows(const HeadRows &a, int t) {
  constexpr int D = LANES * 8, ROWS = 256 / LANES;
  __shared__ __attribute__((aligned(16))) float cosines[kMaxHalf], sines[kMaxHalf];
  const int tid = threadIdx.x, lane = tid % LANES, half = a.half;
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

  int position = 0;
  int64_t to = 0;
  if constexpr (PAGED) {
    const TokenPlace of = find_token(a, t);
    if (of.s < 0) {  // a row of no sequence
      for (int r = r0; r < a.q_heads; r += ROWS) {
        uint16_t *dst = a.q_out + ((int64_t)t * a.q_heads + r) * D;
        *reinterpret_cast<uint2 *>(dst + lo) = *reinterpret_cast<uint2 *>(dst + hi) = uint2{0, 0};
      }
      return;
    }
    position = of.position;
    if (a.k_heads) {  // offset of the token's row of head 0 in the cache; negative: none
      const int64_t room = (int64_t)a.batch.table_pages << a.batch.page_shift;
      to = position < 0 || position >= room
               ? -1
               : paged_page(a.batch, of.s, position) +
                     (int64_t)(position & ((1 << a.batch.page_shift) - 1)) * D;
    }
  }
  if (tid < half) turn(a, freq, tid, t, position, &sines[tid], &cosines[tid]);
  __syncthreads();

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

template <typename T, int LANES, bool PAGED>
__global__ __launch_bounds__(256) void head_rows_kernel(HeadRows a) {
  token_rows<T, LANES, PAGED>(a, blockIdx.x);
}

// ------------------------------------------------------------------ a cache in 8 bits
// Four waves (two for heads of 64) take one side (keys or values) of one head of a block of 16
// positions, as far as the call writes them, in registers: norm, rotation, then the block's largest
// value m and its scale
//   2^e,  e the least with m <= 448 2^e,
// not below that of the rows which the block holds already: a row is rounded again only when a later
// one raises the scale, and as the scale is a power of two, four significant bits stay what they
// were but for values below 2^-6 of it.  Straight from fp32, so a value is rounded once.
// (int8 under such scales would be rounded again in every row whenever one grows.)
//
// Blocks come first, as their chain is the longest: lengths, then page and rows, then the exchange
// of the largest value; the queries' rows go as without a cache, a workgroup a token.  From memory,
// 20 heads of 256 (16 of them queries'): 64 tokens 4.7 us, 4096 tokens 21.6 us (79.7 MB, 3.7 TB/s;
// 19.0 us with the rows in the caches), 16000 64.6 us (4.8 TB/s); 3310 tokens, 48 heads of 128,
// 20.7 us (74.6 MB, 3.6 TB/s; 18.8).  The next side's rows
// requested before the one at hand cost registers and gained nothing; the blocks' workgroups spread
// among the queries' were slower.
struct E4m3Pages {
  uint8_t *k, *v;
  float *scales;
  int64_t scale_stride;
  int shares;  // workgroups of a block, which share its heads' sides
  int blocks;  // workgroups of blocks in all, before those of the queries' tokens
};

// Positions of a sequence that the call writes.
struct Written {
  int first, end;  // positions; first >= end: none
  int row;         // of `first`
};
__device__ __forceinline__ Written written(const HeadRows &a, const PagedSequence &q) {
  const int room = a.batch.table_pages << a.batch.page_shift;
  const int first = max(q.base, 0);
  return {first, (int)min((int64_t)q.base + q.count, (int64_t)room), q.first + first - q.base};
}
__device__ __forceinline__ int block_count(const HeadRows &a, const PagedSequence &q) {
  const Written w = written(a, q);
  return w.first < w.end ? (w.end - 1) / kScaleKeys - w.first / kScaleKeys + 1 : 0;
}

// Sequence of the index-th block of all, and the block's place there; s < 0: none.  All 256 threads.
struct BlockPlace {
  int s, block;
};
__device__ BlockPlace find_block(const HeadRows &a, int index, PagedSequence &seq) {
  __shared__ int sums[4];
  __shared__ BlockPlace found;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = a.batch.sequences;
  if (S <= 64) {  // each wave for itself
    const PagedSequence mine = paged_sequences(a.batch, min(lane, S - 1), a.tokens);
    const int n = lane < S ? block_count(a, mine) : 0, sum = (int)wave_scan((uint32_t)n);
    const uint64_t hit = __ballot(index >= sum - n && index < sum);
    if (!hit) return {-1, 0};
    const int at = __builtin_ctzll(hit);
    seq = sequence_at(a.batch, at, mine, a.tokens);
    return {at, index - __builtin_amdgcn_readlane(sum - n, at)};
  }
  if (tid == 0) found = {-1, 0};
  int64_t base = 0;
  for (int c = 0; c < S && base <= index; c += 256) {
    const PagedSequence mine = paged_sequences(a.batch, min(c + tid, S - 1), a.tokens);
    const int n = c + tid < S ? block_count(a, mine) : 0, sum = (int)wave_scan((uint32_t)n);
    __syncthreads();
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    int64_t before = base + sum - n;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before += sums[w];
      base += sums[w];
    }
    if (index >= before && index < before + n) found = {c + tid, (int)(index - before)};
  }
  __syncthreads();
  if (found.s >= 0) seq = sequence_at(a.batch, found.s, {}, a.tokens);
  return found;
}

// Four values of 8 bits, NaN for what is not finite.
__device__ __forceinline__ uint32_t to_e4m3(const float x[4], float inverse) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * inverse, x[1] * inverse, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * inverse, x[3] * inverse, w, true);
}
// Four held values under a scale 1 / `ratio` times as large.
__device__ __forceinline__ uint32_t rescale_e4m3(uint32_t w, float ratio) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  const float x[4] = {lo[0], lo[1], hi[0], hi[1]};
  return to_e4m3(x, ratio);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

template <typename T, int LANES>
__device__ __forceinline__ void block_rows(const HeadRows &a, const E4m3Pages &p, int index) {
  constexpr int D = LANES * 8, ROWS = 64 / LANES;  // rows of a wave at a time
  constexpr int WAVES = LANES == 8 ? 2 : 4, UNITS = 4 / WAVES;  // of a side, sides at a time
  constexpr int PASSES = kScaleKeys / WAVES / ROWS;
  __shared__ __attribute__((aligned(16))) float cosines[kScaleKeys][kMaxHalf],
      sines[kScaleKeys][kMaxHalf];
  __shared__ int largest[2][4];  // exponents, of the sides in turn
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid % LANES;
  const int row = wave % WAVES * (PASSES * ROWS) + (tid & 63) / LANES;  // of the block, first pass
  PagedSequence seq;
  const BlockPlace at = find_block(a, index / p.shares, seq);
  if (at.s < 0) return;
  const Written w = written(a, seq);
  const int block = w.first / kScaleKeys + at.block, p0 = max(block * kScaleKeys, w.first);
  const int p1 = min((block + 1) * kScaleKeys, w.end);
  const int before = p0 - block * kScaleKeys, count = p1 - p0;  // rows held already, new ones
  const int row0 = w.row + p0 - w.first;                        // of the block's first new position
  const int page = paged_number(a.batch, at.s, p0), nb = 1 << (a.batch.page_shift - kScaleShift);
  const int inside = block & (nb - 1), share = index % p.shares;
  struct Side {  // of a head, and how a lane's channels lie there
    int head, lo, hi;
    bool value, rotated;
  };
  auto side = [&](int first) {
    const int unit = first + wave / WAVES;  // `first` is even where a workgroup has two at a time
    const bool value = unit >= a.k_heads, rotated = !value && lane * 8 < 2 * a.half;
    return Side{value ? unit - a.k_heads : unit, rotated ? lane * 4 : lane * 8,
                rotated ? a.half + lane * 4 : lane * 8 + 4, value, rotated};
  };
  auto load = [&](const Side &d, Row8 (&raw)[PASSES]) {
    const uint16_t *src = d.value ? a.v + d.head * a.v_head : a.k + d.head * a.k_head;
    const int64_t stride = d.value ? a.v_token : a.k_token;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = min(max(row + i * ROWS - before, 0), count - 1);
      const uint16_t *x = src + (row0 + r) * stride;
      raw[i] = Row8{ldg_u2(x + d.lo), ldg_u2(x + d.hi)};
    }
  };
  const int step = p.shares * UNITS;
  if (share * UNITS < a.k_heads) {  // keys among the workgroup's, which come first
    for (int i = tid; i < count * a.half; i += 256) {
      const int r = i / a.half, j = i % a.half;
      turn(a, a.inv_freq[j], j, row0 + r, p0 + r, &sines[r][j], &cosines[r][j]);
    }
    __syncthreads();
  }
  for (int first = share * UNITS, odd = 0; first < 2 * a.k_heads; first += step, odd ^= 1) {
    const Side d = side(first);
    const int head = d.head, lo = d.lo, hi = d.hi;
    const bool value = d.value, rotated = d.rotated;
    Row8 raw[PASSES];
    load(d, raw);
    float *scale = p.scales + page * p.scale_stride + (2 * head + value) * nb + inside;
    // The exponent of the rows held already is the one that attention reads; another program may
    // have left them one below the least, under which they are rounded again.
    int least = kScaleLeast<T>, held = least;
    if (before > 0) {
      held = min((int)(__float_as_uint(*scale) >> 23 & 0xFFu) - 127, kScaleMost<T>);
      least = max(held, least);
    }
    const float *weight = value ? nullptr : a.k_w;
    float w0[4] = {}, w1[4] = {};
    if (weight) {
      *reinterpret_cast<float4 *>(w0) = *reinterpret_cast<const float4 *>(weight + lo);
      *reinterpret_cast<float4 *>(w1) = *reinterpret_cast<const float4 *>(weight + hi);
    }

    float x[PASSES][8], most = 0.0f;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      float *u = x[i], *v = x[i] + 4;
      unpack4<T>(raw[i].lo, u);
      unpack4<T>(raw[i].hi, v);
      if (weight) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(u[j], u[j], ss);
        const float n = 1.0f / sqrtf(lanes_sum<LANES>(ss) * (1.0f / D) + a.eps);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] *= n * (1.0f + w0[j]), v[j] *= n * (1.0f + w1[j]);
      }
      const int r = row + i * ROWS - before;
      if (rotated) {
        const int of = min(max(r, 0), count - 1);
        float c[4], s[4];
        *reinterpret_cast<float4 *>(c) = *reinterpret_cast<const float4 *>(&cosines[of][lo]);
        *reinterpret_cast<float4 *>(s) = *reinterpret_cast<const float4 *>(&sines[of][lo]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float y = u[j] * c[j] - v[j] * s[j];
          v[j] = v[j] * c[j] + u[j] * s[j];
          u[j] = y;
        }
      }
      float top = 0.0f;  // fmaxf passes over NaN
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(u[j]));
      if (r >= 0 && r < count) most = fmaxf(most, top);
    }
    if (__builtin_expect(__any(most > kHeldMost<T>), 0)) {  // and over infinities
      most = 0.0f;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int r = row + i * ROWS - before;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float size = fabsf(x[i][j]);
          x[i][j] = size < INFINITY ? fminf(fmaxf(x[i][j], -kHeldMost<T>), kHeldMost<T>) : NAN;
          if (r >= 0 && r < count && size < INFINITY) most = fmaxf(most, fabsf(x[i][j]));
        }
      }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    // 448 = 1.75 * 2^8: one more where the significand is above 1.75
    int e = max((int)((__float_as_uint(most) + 0x1FFFFFu) >> 23) - 127 - 8, least);
    if ((tid & 63) == 0) largest[odd][wave] = e;
    __syncthreads();  // every wave has read the scale
#pragma unroll
    for (int i = 0; i < WAVES; ++i) e = max(e, largest[odd][wave / WAVES * WAVES + i]);
    uint8_t *rows = (value ? p.v : p.k) + page * a.batch.page_stride +
                    (((int64_t)head << a.batch.page_shift) + inside * kScaleKeys) * D;
    const float inverse = power_of_two(-e), ratio = power_of_two(max(held - e, -126));
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int r = row + i * ROWS;
      if (r < before) {
        if (e > held) {
          uint2 *b = reinterpret_cast<uint2 *>(rows + r * D + lane * 8);
          const uint2 old = *b;
          *b = uint2{rescale_e4m3(old.x, ratio), rescale_e4m3(old.y, ratio)};
        }
      } else if (r < before + count) {
        *reinterpret_cast<uint32_t *>(rows + r * D + lo) = to_e4m3(x[i], inverse);
        *reinterpret_cast<uint32_t *>(rows + r * D + hi) = to_e4m3(x[i] + 4, inverse);
      }
    }
    if (tid % (WAVES * 64) == 0) *scale = power_of_two(e);
  }
}

template <typename T, int LANES>
__global__ __launch_bounds__(256) void append_e4m3_kernel(HeadRows a, E4m3Pages p) {
  if (blockIdx.x < p.blocks) {
    block_rows<T, LANES>(a, p, blockIdx.x);
  } else {
    a.k_heads = 0;
    token_rows<T, LANES, true>(a, blockIdx.x - p.blocks);
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

// Checks of positions and the axes of the pairs; positions may be missing with a cache.
int check_axes(const int64_t *positions, int64_t position_stride, int64_t axes,
               const int32_t *axis, int64_t tokens) {
  LM_REQUIRE(axes >= 1 && axes <= 64, LM_EINVAL, "invalid number of axes");
  LM_REQUIRE(!axis || positions, LM_EINVAL, "axes need positions");
  LM_REQUIRE(axes == 1 || position_stride >= tokens, LM_EINVAL, "positions of the axes overlap");
  return LM_OK;
}

int norm_rope(const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads,
              const float *q_weight, void *q_out, const void *k, int64_t k_token_stride,
              int64_t k_head_stride, int64_t k_heads, const float *k_weight, void *k_out,
              const int64_t *positions, int64_t position_stride, int64_t axes, const int32_t *axis,
              const float *inv_freq, int64_t pairs, int64_t tokens, int64_t head_dim, float eps,
              int dtype, void *stream) {
  LM_REQUIRE(dtype == LM_BF16 || dtype == LM_FP16, LM_EINVAL, "attention requires FP16/BF16");
  LM_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, LM_EINVAL,
             "attention supports heads of 64, 128 or 256");
  LM_REQUIRE(q_heads >= 0 && q_heads <= 65536 && k_heads >= 0 && k_heads <= 65536, LM_EINVAL,
             "invalid number of heads");
  LM_REQUIRE(tokens >= 0 && tokens < kMaxTokens, LM_EINVAL, "invalid token count");
  if (const int rc = check_rotation(inv_freq, pairs, head_dim)) return rc;
  if (tokens == 0 || q_heads + k_heads == 0) return LM_OK;
  if (const int rc = check_axes(positions, position_stride, axes, axis, tokens)) return rc;
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
  a.positions = positions, a.position_stride = position_stride;
  a.axis = axis, a.axes = (int)axes, a.inv_freq = inv_freq, a.half = (int)pairs;
  a.tokens = (int)tokens, a.eps = eps;
  if (dtype == LM_BF16)
    launch_rows<BF16, false>(a, (int)head_dim, as_stream(stream));
  else
    launch_rows<FP16, false>(a, (int)head_dim, as_stream(stream));
  return check_launch("head_rows_kernel");
}

template <typename T>
void launch_e4m3(const HeadRows &a, const E4m3Pages &p, int head_dim, hipStream_t st) {
  const unsigned grid = (unsigned)(p.blocks + (a.q_heads ? a.tokens : 0));
  if (head_dim == 256)
    append_e4m3_kernel<T, 32><<<grid, 256, 0, st>>>(a, p);
  else if (head_dim == 128)
    append_e4m3_kernel<T, 16><<<grid, 256, 0, st>>>(a, p);
  else
    append_e4m3_kernel<T, 8><<<grid, 256, 0, st>>>(a, p);
}

// An append to a cache of the rows' type, or of 8 bits (e4m3).
int paged_append(const void *k, int64_t k_token_stride, int64_t k_head_stride,
                 const float *k_weight, const void *v, int64_t v_token_stride,
                 int64_t v_head_stride, const void *q, int64_t q_token_stride,
                 int64_t q_head_stride, int64_t q_heads, const float *q_weight, void *q_out,
                 void *k_pages, void *v_pages, bool e4m3, float *scales, int64_t scale_stride,
                 int64_t pages, int64_t page_stride, int64_t kv_heads, int64_t page_size,
                 int64_t head_dim, const int32_t *starts, const int32_t *lengths,
                 const int32_t *table, int64_t table_stride, int64_t table_pages,
                 int64_t sequences, const int64_t *positions, int64_t position_stride,
                 int64_t axes, const int32_t *axis, const float *inv_freq, int64_t pairs,
                 int64_t tokens, float eps, int dtype, void *stream) {
  if (const int rc = paged_check(pages, page_stride, kv_heads, page_size, head_dim, starts, lengths,
                                 table, table_stride, table_pages, sequences, tokens, dtype))
    return rc;
  LM_REQUIRE(q_heads >= 0 && q_heads <= 65536, LM_EINVAL, "invalid number of heads");
  if (const int rc = check_rotation(inv_freq, pairs, head_dim)) return rc;
  if (const int rc = check_axes(positions, position_stride, axes, axis, tokens)) return rc;
  const bool empty = tokens == 0 || sequences == 0;
  if (e4m3)
    if (const int rc = scales_check(scales, scale_stride, kv_heads, page_size, page_stride, empty))
      return rc;
  if (empty) return LM_OK;
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
  a.batch = {starts, lengths, table, table_stride, (int)sequences, (int)table_pages,
             __builtin_ctzll((unsigned long long)page_size), (int)pages, page_stride,
             (int)kv_heads};
  a.positions = positions, a.position_stride = position_stride;
  a.axis = axis, a.axes = (int)axes, a.inv_freq = inv_freq, a.half = (int)pairs;
  a.tokens = (int)tokens, a.eps = eps;
  if (e4m3) {
    E4m3Pages p = {static_cast<uint8_t *>(k_pages), static_cast<uint8_t *>(v_pages), scales,
                   scale_stride, 1, 0};
    // n positions of a sequence lie in at most n / 16 + 2 blocks, and in n of them
    const int64_t bound = tokens / kScaleKeys + 2 * sequences, most = bound < tokens ? bound : tokens;
    // Four workgroups a CU, if the sides are that many: with half or twice as many, 9 sequences of 30
    // to 900 tokens (32 + 8 heads of 128) took 19.5 and 21.5 us instead of 19.3, 4 of 700 (16 + 16
    // heads of 64) 16.5 and 14.5 instead of 13.1.
    const int64_t sides = head_dim == 64 ? kv_heads : 2 * kv_heads, some = 1024 / most;
    p.shares = (int)(some < 1 ? 1 : some < sides ? some : sides);
    LM_REQUIRE(most * p.shares + tokens < (1LL << 24), LM_EINVAL, "too many rows");
    p.blocks = (int)(most * p.shares);
    if (dtype == LM_BF16)
      launch_e4m3<BF16>(a, p, (int)head_dim, as_stream(stream));
    else
      launch_e4m3<FP16>(a, p, (int)head_dim, as_stream(stream));
    return check_launch("append_e4m3_kernel");
  }
  a.k_pages = static_cast<uint16_t *>(k_pages), a.v_pages = static_cast<uint16_t *>(v_pages);
  if (dtype == LM_BF16)
    launch_rows<BF16, true>(a, (int)head_dim, as_stream(stream));
  else
    launch_rows<FP16, true>(a, (int)head_dim, as_stream(stream));
  return check_launch("head_rows_kernel");
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
  return norm_rope(q, q_token_stride, q_head_stride, q_heads, q_weight, q_out, k, k_token_stride,
                   k_head_stride, k_heads, k_weight, k_out, positions, 0, 1, nullptr, inv_freq,
                   pairs, tokens, head_dim, eps, dtype, stream);
}

extern "C" int lm_qk_norm_rope_axes(const void *q, int64_t q_token_stride, int64_t q_head_stride,
                                    int64_t q_heads, const float *q_weight, void *q_out,
                                    const void *k, int64_t k_token_stride, int64_t k_head_stride,
                                    int64_t k_heads, const float *k_weight, void *k_out,
                                    const int64_t *positions, int64_t position_stride,
                                    int64_t axes, const int32_t *axis, const float *inv_freq,
                                    int64_t pairs, int64_t tokens, int64_t head_dim, float eps,
                                    int dtype, void *stream) {
  return norm_rope(q, q_token_stride, q_head_stride, q_heads, q_weight, q_out, k, k_token_stride,
                   k_head_stride, k_heads, k_weight, k_out, positions, position_stride, axes, axis,
                   inv_freq, pairs, tokens, head_dim, eps, dtype, stream);
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
  return paged_append(k, k_token_stride, k_head_stride, k_weight, v, v_token_stride, v_head_stride,
                      q, q_token_stride, q_head_stride, q_heads, q_weight, q_out, k_pages, v_pages,
                      false, nullptr, 0, pages, page_stride, kv_heads, page_size, head_dim, starts,
                      lengths, table, table_stride, table_pages, sequences, nullptr, 0, 1, nullptr,
                      inv_freq, pairs, tokens, eps, dtype, stream);
}

extern "C" int lm_paged_append_axes(
    const void *k, int64_t k_token_stride, int64_t k_head_stride, const float *k_weight,
    const void *v, int64_t v_token_stride, int64_t v_head_stride, const void *q,
    int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads, const float *q_weight,
    void *q_out, void *k_pages, void *v_pages, int64_t pages, int64_t page_stride,
    int64_t kv_heads, int64_t page_size, int64_t head_dim, const int32_t *starts,
    const int32_t *lengths, const int32_t *table, int64_t table_stride, int64_t table_pages,
    int64_t sequences, const int64_t *positions, int64_t position_stride, int64_t axes,
    const int32_t *axis, const float *inv_freq, int64_t pairs, int64_t tokens, float eps, int dtype,
    void *stream) {
  return paged_append(k, k_token_stride, k_head_stride, k_weight, v, v_token_stride, v_head_stride,
                      q, q_token_stride, q_head_stride, q_heads, q_weight, q_out, k_pages, v_pages,
                      false, nullptr, 0, pages, page_stride, kv_heads, page_size, head_dim, starts,
                      lengths, table, table_stride, table_pages, sequences, positions,
                      position_stride, axes, axis, inv_freq, pairs, tokens, eps, dtype, stream);
}

extern "C" int lm_paged_append_e4m3(
    const void *k, int64_t k_token_stride, int64_t k_head_stride, const float *k_weight,
    const void *v, int64_t v_token_stride, int64_t v_head_stride, const void *q,
    int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads, const float *q_weight,
    void *q_out, void *k_pages, void *v_pages, float *scales, int64_t scale_stride, int64_t pages,
    int64_t page_stride, int64_t kv_heads, int64_t page_size, int64_t head_dim,
    const int32_t *starts, const int32_t *lengths, const int32_t *table, int64_t table_stride,
    int64_t table_pages, int64_t sequences, const int64_t *positions, int64_t position_stride,
    int64_t axes, const int32_t *axis, const float *inv_freq, int64_t pairs, int64_t tokens,
    float eps, int dtype, void *stream) {
  return paged_append(k, k_token_stride, k_head_stride, k_weight, v, v_token_stride, v_head_stride,
                      q, q_token_stride, q_head_stride, q_heads, q_weight, q_out, k_pages, v_pages,
                      true, scales, scale_stride, pages, page_stride, kv_heads, page_size, head_dim,
                      starts, lengths, table, table_stride, table_pages, sequences, positions,
                      position_stride, axes, axis, inv_freq, pairs, tokens, eps, dtype, stream);
}
