// Attention of each sequence's new tokens over its paged cache (gfx950).
//
//   o_t = sum_{j <= p_t} e^{x_j - m} v_j / sum_j e^{x_j - m},   x_j = scale q_t . k_j
//
// causal at the end of the sequence, times sigmoid(gate_t) where a gate is given;
// a row without a visible key is 0.  One pass over the keys with a running m and
// sum (exponentials in base 2, fp32); m follows the maximum (in fp16 2^kLift below
// it) only when that has grown by more than 2^kSlack, so the accumulated rows are
// rarely rescaled.
//
// Both kernels form the transposed products.  S^T = K Q^T leaves a lane with one
// query (its column) and a few consecutive keys, so a column's statistics are the
// lane's own, and the weights are already the operand of O^T = V^T P^T: the keys
// of a lane's C registers are the k indices its operand registers hold.  V^T comes
// from the row-major V tile by the LDS transpose read, four keys of one channel a
// lane.  K and V go from the cache into LDS by direct loads, whole rows at a time,
// the 16-byte pieces of a row permuted (swizzle) so that neither read meets a bank
// conflict.  The weights are rounded to the inputs' type for the second product, as
// the matrix cores take both operands of one type and a second product for what the
// rounding leaves would double it; their sum is of the unrounded ones in fp32, and
// the result is rounded once.  Against 64 bits a result is off by 0.0018 to 0.0023
// of the norm in bf16 and 0.00026 in fp16; its own rounding alone is 0.0017 and
// 0.00021 of that.
//
//  attention_few_kernel   sequences of at most 16 rows (new tokens x query heads of
//                         a key-value head): bound by the cache's bytes.  16-column
//                         tiles; the keys of all such sequences, one after another,
//                         are cut into equal spans, a workgroup each, and the four
//                         waves of a workgroup take 16 keys of it in turn, each with
//                         a ring of its own in LDS, so nothing waits for another
//                         wave.  Times on one MI355X, heads of 256 and 2 key-value
//                         heads: 262144 keys of one sequence 88 us (6.1 TB/s), 64
//                         sequences of 400 to 13000 keys 92 us (5.8 TB/s); 16 heads
//                         of 64, 24 sequences of 300 to 5000 keys with 2 to 9 rows
//                         29 us (5.3 TB/s).
//  attention_tile_kernel  longer ones: bound by the matrix cores and the softmax
//                         beside them.  128 rows a workgroup, 32 a wave.  Heads of
//                         256 leave a wave no registers for a second one of its kind
//                         on a SIMD unless both work for the same rows: eight waves,
//                         two key groups, on shared 64-key tiles; smaller heads have
//                         four waves on 32-key tiles.  Two tiles in LDS, one read
//                         and one loaded.  Few tiles split their keys over workgroups
//                         too.  2048 tokens of 16 heads of 256 (2 key-value heads)
//                         behind 8192 keys: 293 to 302 us in a long run of calls,
//                         1024 to 1054 TFLOP/s (1371 for a large library product);
//                         without a history 64 us.
//  attention_combine_kernel  joins the parts of split keys, 4 to 12 us: the partial
//                         sums are fp32, written and read once.
#include <cmath>
#include <utility>

#include "paged.hpp"

namespace lm {
namespace {

#define LDS __attribute__((address_space(3)))
#define GLB __attribute__((address_space(1)))

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// The parts of a sequence at a key-value head: their first span, its place there, their count.
struct Parts {
  int span, later, count;
};

struct Attention {
  const uint16_t *q, *gate;  // gate: null or a row for each row of q
  int64_t q_token, q_head, gate_token, gate_head;  // strides, elements
  const uint16_t *k_pages, *v_pages;
  uint16_t *out;  // [tokens][q_heads][D]
  float *part, *part_ml;  // few: unscaled sums of split keys, and (m, l) of each row
  float *tile_part, *tile_ml;  // the same of tiles
  Parts *parts;   // few: [sequences][kv_heads]
  PagedBatch batch;
  int tokens, q_heads, group;
  int shares;  // few: spans that a key-value head's keys are cut into, at most
  int splits;  // tile: parts of a tile's keys, at most
  int room;    // tile: workgroups at a time for a key-value head, 0: every tile has `splits` parts
  int *row_parts;  // tile, if room > 0: parts of each row, [tokens][q_heads]
  bool few;    // tile: sequences of few rows are attention_few_kernel's
  float scale2;   // |scale| * log2(e), not 0
  uint32_t flip;  // sign bits that queries are flipped by, for a negative scale
};

constexpr int kFewRows = 16;    // columns of the few-row kernel
constexpr float kSlack = 8.0f;  // weights stay below 2^(8 + kLift)
// How far m stays below the maximum.  fp16 ends at 2^-24: with weights of at most 1 a tail of keys
// 2^-25 below one of them is lost from the products, but not from the sum of the weights; 2^7 more
// keeps it to 2^-32, and the largest weight at 2^15, finite in fp16.  bf16 has fp32's exponents.
template <typename T>
constexpr float kLift = __is_same(T, FP16) ? 7.0f : 0.0f;

__device__ __forceinline__ f32x4 mfma16(BF16, u32x4 a, u32x4 b, f32x4 c) {
  return BF16::mfma16x16x32(a, b, c);
}
__device__ __forceinline__ f32x4 mfma16(FP16, u32x4 a, u32x4 b, f32x4 c) {
  return FP16::mfma16x16x32(a, b, c);
}
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma16k16(BF16, u32x2 a, u32x2 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a),
                                                   __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16k16(FP16, u32x2 a, u32x2 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a),
                                               __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(BF16, u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(FP16, u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Exchanges between the 16-lane rows (xor 16) and the halves (xor 32) of a wave.
template <typename F>
__device__ __forceinline__ float across16(float v, F f) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <typename F>
__device__ __forceinline__ float across32(float v, F f) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Add {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
// 2^(m - n) of two running maxima, n >= m; both may be -inf.
__device__ __forceinline__ float decay(float m, float n) { return m == n ? 1.0f : exp2_hw(m - n); }

// Piece c (16 bytes) of row r of a tile lies at place c ^ swizzle(r) of the row, so that the
// rows that one LDS read touches use different banks (a row is D * 2 bytes, the banks repeat
// every 256).  kRows: reads of one or two pieces of 16 rows; kQuads: of four pieces of 4 rows
// (the transpose reads of 32 channels; with kRows they took 4 times as long).  Linear over
// disjoint bits of r: a read's lane part is formed once, its constant part is one exclusive or.
enum Swizzle { kRows, kQuads };
template <int D, Swizzle S = kRows>
__device__ __forceinline__ constexpr int swizzle(int r) {
  return S == kRows ? (D == 64 ? (r >> 1) & 7 : r & 15) : (D == 64 ? (r & 2) << 1 : (r & 3) << 2);
}

// Cache policy of loads that are not read again (non-temporal): 262144 keys of one sequence
// in 88 us instead of 96; the tiles, which other workgroups read too, take 10 % longer with it.
constexpr int kStream = 2;

// ROWS rows of a page, from `src` (row `row0` of the tile), into LDS: wave-wide loads of
// 1 KB, lane-linear in LDS, so the swizzle permutes the source.  Rows behind a sequence's
// end are loaded as they are (their page holds them) and masked later.  An instruction's
// offset counts for both addresses, so four share a pair of them.
template <int D, int PER, Swizzle S, int POLICY, int... I>
__device__ __forceinline__ void load_4k(const GLB char *from, uint32_t off, int row0, LDS char *to,
                                        std::integer_sequence<int, I...>) {
  (__builtin_amdgcn_global_load_lds(
       (const GLB void *)(from + (off ^ (swizzle<D, S>(row0 + I * PER) << 4))), (LDS void *)to, 16,
       I * 1024, POLICY),
   ...);
}
template <int D, int ROWS, Swizzle S = kRows, int POLICY = 0>
__device__ __forceinline__ void load_rows(const uint16_t *src, int row0, LDS char *to, int lane) {
  constexpr int PIECES = D / 8, PER = 64 / PIECES, LOADS = ROWS / PER, GROUP = LOADS < 4 ? LOADS : 4;
  const int own = lane / PIECES;
  const uint32_t off = own * (D * 2) + (((lane % PIECES) ^ swizzle<D, S>(own)) << 4);
#pragma unroll
  for (int i = 0; i < LOADS / GROUP; ++i)
    load_4k<D, PER, S, POLICY>((const GLB char *)src + i * 4096, off, row0 + i * 4 * PER, to + i * 4096,
                       std::make_integer_sequence<int, GROUP>{});
}

// Has v loaded here, so that no wait for it is placed in a loop over direct loads, where it
// would wait for those too.
template <typename V>
__device__ __forceinline__ void settle(V &v) {
  asm volatile("" : "+v"(v));
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Four keys of one channel, by the LDS transpose read: lane i of each 16 lanes gets channel
// d0 + i of rows r .. r + 3, r = row + ROW and d0 = d + CH with the lane's own row (a multiple
// of 4) and d (0 or 16) in `base` (transpose_base), the rest constant.
template <int D, Swizzle S>
__device__ __forceinline__ int transpose_base(int row, int d, int lane) {
  const int r = row + (lane & 15) / 4;
  return r * (D * 2) + (((d / 8 + (lane & 3) / 2) ^ swizzle<D, S>(r)) << 4) + (lane & 1) * 8;
}
// The address of piece `ch` (constant) of row `row` (constant) past a lane's base, in which
// the piece's low four bits were swizzled.
template <int D, Swizzle S>
__device__ __forceinline__ int swizzled(int base, int row, int ch) {
  return (base ^ (((ch & 15) ^ swizzle<D, S>(row)) << 4)) + (ch & 16) * 16 + row * (D * 2);
}
template <int D, Swizzle S>
__device__ __forceinline__ u32x2 read_transposed(const LDS char *tile, int base, int row, int d) {
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                 (LDS s16x4 *)(tile + swizzled<D, S>(base, row, d / 8))));
}

// Eight or four such reads at once, waited for here: before the builtin's read the compiler waits
// for every direct load in flight, which emptied the few-row kernel's rings at each step (24
// sequences of 300 to 5000 keys, 16 heads of 64: 33 us instead of 37, 64 of 400 to 13000 keys, 8
// heads of 128: 127 instead of 134).  The tiles keep the builtin: their loads are due by then,
// and reads waited for in groups took 4 % more there.
template <int OFFSET>
__device__ __forceinline__ void read_transposed8(u32x2 (&v)[8], const LDS char *const (&at)[8]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%16\n\tds_read_b64_tr_b16 %1, %9 offset:%16\n\t"
      "ds_read_b64_tr_b16 %2, %10 offset:%16\n\tds_read_b64_tr_b16 %3, %11 offset:%16\n\t"
      "ds_read_b64_tr_b16 %4, %12 offset:%16\n\tds_read_b64_tr_b16 %5, %13 offset:%16\n\t"
      "ds_read_b64_tr_b16 %6, %14 offset:%16\n\tds_read_b64_tr_b16 %7, %15 offset:%16\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]),
        "=&v"(v[6]), "=&v"(v[7])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]),
        "v"(at[7]), "n"(OFFSET)
      : "memory");
}
__device__ __forceinline__ void read_transposed4(u32x2 (&v)[4], const LDS char *const (&at)[4]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %5\n\t"
      "ds_read_b64_tr_b16 %2, %6\n\tds_read_b64_tr_b16 %3, %7\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
      : "memory");
}

// Keeps a lane's base from being expanded into one register for every constant part.
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Values of keys that some row does not see: a weight of 0 must not meet an infinity or
// NaN (0 * inf).  The products of such keys take the finite values, 0 for others, and where
// there were others, the rows that do see the key get them added afterwards.
template <typename T>
struct Pair {
  static constexpr uint32_t E = __is_same(T, BF16) ? 0x7F80u : 0x7C00u;     // infinity
  static constexpr uint32_t STEP = 0x8000u - E;  // carries it, and NaN, into the sign bit
  static __device__ __forceinline__ uint32_t odd(uint32_t v) {  // sign bits set where odd
    return (v & 0x7FFF7FFFu) + (STEP | STEP << 16);
  }
  static __device__ __forceinline__ uint32_t finite(uint32_t v, uint32_t &any) {
    const uint32_t s = odd(v) & 0x80008000u;
    any |= s;
    return v & ~(s | (s - (s >> 15)));  // all bits of the halves where odd
  }
  static __device__ __forceinline__ float odd_part(uint32_t x) {
    return (x & E) == E ? T::to_f32(x) : 0.0f;
  }
};

// The infinities and NaN among four channels, 0 for others.
template <typename T>
__device__ __forceinline__ f32x4 odd_parts(const uint16_t *v) {
  const uint2 w = ldg_u2(v);
  return f32x4{Pair<T>::odd_part(w.x & 0xFFFFu), Pair<T>::odd_part(w.x >> 16),
               Pair<T>::odd_part(w.y & 0xFFFFu), Pair<T>::odd_part(w.y >> 16)};
}

// Value row of key k of sequence s at the key-value head whose rows begin at `head`.
template <int D>
__device__ __forceinline__ const uint16_t *value_row(const Attention &a, int s, int64_t head, int k) {
  return a.v_pages + paged_page(a.batch, s, k) + head +
         (int64_t)(k & ((1 << a.batch.page_shift) - 1)) * D;
}

// ------------------------------------------------------------------ shares of keys
// The keys of the sequences with few rows, in blocks of 64 and one sequence after another,
// are cut into `shares` equal spans, one for each workgroup of a key-value head: as much
// work for each, whatever the lengths.  Every workgroup works the cuts out from the lengths,
// so the host needs to know none of them and a captured call follows them.
constexpr int kBlockKeys = 64;

// count > 0 of a sequence whose rows fit the few-row kernel
__device__ __forceinline__ bool few_rows(const PagedSequence &q, int group) {
  return q.count > 0 && q.count <= kFewRows / group;
}
// Blocks of sequence s: 0 of one that is not the few-row kernel's, at least 1 of others.
__device__ __forceinline__ int few_blocks(const Attention &a, int s) {
  if (s >= a.batch.sequences) return 0;
  const PagedSequence q = paged_sequence(a.batch, s, a.tokens);
  return few_rows(q, a.group) ? max((q.length + kBlockKeys - 1) / kBlockKeys, 1) : 0;
}

struct Spans {
  int64_t blocks;  // of all sequences
  int spans;       // at most `blocks`
  __device__ __forceinline__ int64_t start(int span) const { return blocks * span / spans; }
  __device__ __forceinline__ int of(int64_t block) const {  // the span that holds a block
    return (int)(((block + 1) * spans - 1) / blocks);
  }
};
struct Find {
  int64_t first;  // of the found sequence: its first block
  int s;          // < 0: none
};

// The spans, and the sequence that holds the first block of span `index`.  All 256 threads;
// scratch (8 words of LDS) and found are free again afterwards.
__device__ Spans find_span(const Attention &a, int index, int64_t *scratch, Find *found, Find &got) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = a.batch.sequences;
  Spans sp;
  got = {0, -1};
  if (S <= 64) {  // every wave by itself: a sequence a lane
    const uint32_t n = few_blocks(a, lane);  // 64 of at most 2^25
    uint32_t sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = __shfl_up(sum, o, 64);
      if (lane >= o) sum += v;
    }
    sp.blocks = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
    sp.spans = (int)min((int64_t)a.shares, sp.blocks);
    if (index < sp.spans) {
      const int64_t want = sp.start(index);
      const int s = __builtin_ctzll(__ballot(want < (int64_t)sum));  // the first that ends after it
      got = {(uint32_t)__builtin_amdgcn_readlane((int)(sum - n), s), s};
    }
    return sp;
  }
  if (tid == 0) found->s = -1;
  const int mine = few_blocks(a, tid);
  int64_t all = mine;
  for (int s = tid + 256; s < S; s += 256) all += few_blocks(a, s);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) all += __shfl_xor(all, o, 64);
  if (lane == 0) scratch[wave] = all;
  __syncthreads();
  sp.blocks = scratch[0] + scratch[1] + scratch[2] + scratch[3];
  sp.spans = (int)min((int64_t)a.shares, sp.blocks);
  if (index < sp.spans) {
    const int64_t want = sp.start(index);
    int64_t base = 0;  // blocks before this group of 256 sequences
    for (int c = 0; c < S && base <= want; c += 256) {
      const int n = c == 0 ? mine : few_blocks(a, c + tid);
      int64_t sum = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int64_t v = __shfl_up(sum, o, 64);
        if (lane >= o) sum += v;
      }
      __syncthreads();
      if (lane == 63) scratch[4 + wave] = sum;
      __syncthreads();
      int64_t before = base + sum - n;
      for (int w = 0; w < 4; ++w) {
        if (w < wave) before += scratch[4 + w];
        base += scratch[4 + w];
      }
      if (n > 0 && want >= before && want < before + n) *found = {before, c + tid};
    }
  }
  __syncthreads();
  got = *found;
  __syncthreads();
  return sp;
}

// ------------------------------------------------------------------ few rows
constexpr int kFewWaves = 4;

// Steps of 16 keys in a wave's ring: 64 KB for a workgroup, two of which share a CU, or 32 KB
// with heads of 64, of which three do: of 24 sequences of 300 to 5000 keys 33 instead of 37 us,
// of 200 up to 1000 keys 69 instead of 77 (16 heads each), one of 100000 keys 25 instead of
// 23.5.  Four workgroups, or three with 48 KB, took 1 to 5 % more than three with 32.
template <int D>
constexpr int few_steps() { return D == 256 ? 1 : 2; }
template <int D>
constexpr int few_ring() { return few_steps<D>() * 2 * 16 * D * 2; }
template <int D>
constexpr int few_merge() { return kFewWaves * (kFewRows * (D + 4) + 2 * kFewRows) * 4; }
template <int D>
constexpr int few_lds() {
  return kFewWaves * few_ring<D>() > few_merge<D>() ? kFewWaves * few_ring<D>() : few_merge<D>();
}

// The running state of a wave's 16 columns (column lane & 15 in each 16 lanes).
template <int D>
struct FewState {
  float m = -INFINITY, l = 0.0f;  // l: this lane's keys only
  f32x4 o[D / 16] = {};           // channels 16 i + 4 (lane >> 4) .. + 3
  bool odd = false;               // infinities or NaN were left out
};

// Products of one 16-key step with the columns: the weights of keys 4 g .. 4 g + 3, packed.
template <typename T, int D>
__device__ __forceinline__ u32x2 few_scores(const LDS char *kt, const u32x4 (&q)[D / 32], int key0,
                                            int limit, float scale2, FewState<D> &st, int lane) {
  const int g = lane >> 4, r = lane & 15;
  const int base = opaque(r * (D * 2) + ((g ^ swizzle<D>(r)) << 4));
  f32x4 s[2] = {};
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const u32x4 k = *(const LDS u32x4 *)(kt + swizzled<D, kRows>(base, 0, i * 4));
    s[i & 1] = mfma16(T{}, k, q[i], s[i & 1]);
  }
  float x[4], mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = key0 + g * 4 + i < limit ? s[0][i] + s[1][i] : -INFINITY;
    mx = fmaxf(mx, x[i]);
  }
  mx = __builtin_fmaf(across32(across16(mx, Max()), Max()), scale2, -kLift<T>);
  if (__any(mx > st.m + kSlack)) {
    const float n = fmaxf(st.m, mx), keep = decay(st.m, n);
    st.m = n;
    st.l *= keep;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) st.o[i] *= keep;
  }
  const float at = st.m == -INFINITY ? 0.0f : st.m;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = exp2_hw(__builtin_fmaf(x[i], scale2, -at));
    st.l += x[i];
  }
  return u32x2{T::pack2(x[0], x[1]), T::pack2(x[2], x[3])};
}

// The values of a 16-key step as operands, 16 channels each.
template <int D>
__device__ __forceinline__ void few_operands(const LDS char *vt, u32x2 (&v)[D / 16], int lane) {
  const int base = opaque(transpose_base<D, kRows>((lane >> 4) * 4, 0, lane));
  constexpr int N = D == 64 ? 4 : 8;
  const LDS char *at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) at[i] = vt + swizzled<D, kRows>(base, 0, i * 2);
  if constexpr (D == 64) {
    read_transposed4(v, at);
  } else {
    read_transposed8<0>(*reinterpret_cast<u32x2(*)[8]>(&v[0]), at);
    if constexpr (D == 256) read_transposed8<256>(*reinterpret_cast<u32x2(*)[8]>(&v[8]), at);
  }
}

// Adds the weighted values of a 16-key step; `mixed`: some row does not see all its keys.
template <typename T, int D>
__device__ __forceinline__ void few_values(const LDS char *vt, u32x2 p, bool mixed,
                                           FewState<D> &st, int lane) {
  u32x2 v[D / 16];
  few_operands<D>(vt, v, lane);
  if (mixed) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      v[i] = u32x2{Pair<T>::finite(v[i][0], any), Pair<T>::finite(v[i][1], any)};
    st.odd |= __any(any != 0);
  }
#pragma unroll
  for (int i = 0; i < D / 16; ++i) st.o[i] = mfma16k16(T{}, v[i], p, st.o[i]);
}

// The keys of a wave: steps of 16 keys, `stride` steps apart, and the pages they lie in.
struct FewKeys {
  const uint16_t *k, *v;  // of the key-value head, in page 0
  const int32_t *table;
  int64_t page_stride;
  int shift, pages, entries;
  int first, stride, steps;  // first step's number, and how many
  int page_of;               // pages of 64 steps, one a lane
};

__device__ __forceinline__ void few_pages(FewKeys &f, int from, int lane) {
  const int step = f.first + min(from + lane, max(f.steps - 1, 0)) * f.stride;
  const int i = min((step * 16) >> f.shift, f.entries - 1);
  f.page_of = clamp_index32(f.table[i], f.pages);
  settle(f.page_of);
}

// Loads step i's rows of one side (a step past the end: again the last, never used).
template <int D>
__device__ __forceinline__ void few_load(const FewKeys &f, const uint16_t *side, int i,
                                         LDS char *to, int lane) {
  const int j = min(i, f.steps - 1), key = (f.first + j * f.stride) * 16;
  const int page = __builtin_amdgcn_readlane(f.page_of, j & 63);
  const uint16_t *src = side + page * f.page_stride + (int64_t)(key & ((1 << f.shift) - 1)) * D;
  load_rows<D, 16, kRows, kStream>(src, 0, to, lane);
}

// Step i, from its place in the ring, which is refilled as soon as it is read; the counts of
// loads that may still be out are stated here.
template <typename T, int D>
__device__ __forceinline__ void few_step(LDS char *ring, const FewKeys &f, const u32x4 (&q)[D / 32],
                                         int i, int limit, int all_see, float scale2,
                                         FewState<D> &st, int lane) {
  constexpr int TILE = 16 * D * 2, N = TILE / 1024;  // bytes and loads of one side of a step
  constexpr int STEPS = few_steps<D>(), OUT = (2 * STEPS - 1) * N;
  LDS char *k = ring + i % STEPS * 2 * TILE, *v = k + TILE;
  const int key = (f.first + i * f.stride) * 16;
  wait_loads<OUT>();
  const u32x2 p = few_scores<T, D>(k, q, key, limit, scale2, st, lane);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  few_load<D>(f, f.k, i + STEPS, k, lane);
  wait_loads<OUT>();
  few_values<T, D>(v, p, key + 16 > all_see, st, lane);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  few_load<D>(f, f.v, i + STEPS, v, lane);
}

// Row c of a sequence's rows at a key-value head: new token c / group, query head
// kv * group + c % group.
struct RowPlace {
  int token, head;
};
__device__ __forceinline__ RowPlace row_place(const Attention &a, const PagedSequence &q, int kv,
                                              int c) {
  return {q.first + c / a.group, kv * a.group + c % a.group};
}

// sigmoid(x) by the hardware's exp2 and reciprocal, off by (1.25 |x| + 5) 2^-24 of it at most: half
// a step of the exponent (1) and the constant log2(e) in fp32 (0.23) count |x| times in e^-x, then
// exp2 (2), the sum (1) and the reciprocal (2).  Results below 2^-126 may be 0.
__device__ __forceinline__ float sigmoid_hw(float x) {
  return __builtin_amdgcn_rcpf(1.0f + exp2_hw(x * -1.4426950408889634f));
}

// Four channels from d of a row's gate, if there is one.
__device__ __forceinline__ uint2 load_gate(const Attention &a, RowPlace at, int d) {
  if (!a.gate) return uint2{0, 0};
  return ldg_u2(a.gate + (int64_t)at.token * a.gate_token + (int64_t)at.head * a.gate_head + d);
}

// Four channels from d of a finished row: gated, rounded once.
template <typename T, int D>
__device__ __forceinline__ void write_row(const Attention &a, RowPlace at, int d, f32x4 o,
                                          uint2 g) {
  if (a.gate) {
    o[0] *= sigmoid_hw(T::to_f32(g.x & 0xFFFFu));
    o[1] *= sigmoid_hw(T::to_f32(g.x >> 16));
    o[2] *= sigmoid_hw(T::to_f32(g.y & 0xFFFFu));
    o[3] *= sigmoid_hw(T::to_f32(g.y >> 16));
  }
  *reinterpret_cast<uint2 *>(a.out + ((int64_t)at.token * a.q_heads + at.head) * D + d) =
      uint2{T::pack2(o[0], o[1]), T::pack2(o[2], o[3])};
}

// Where a span's part of a sequence goes, when it is not all of the sequence: place 0 of the
// span for its first part, 1 for a later one (its last).
__device__ __forceinline__ int64_t part_row(const Attention &a, int span, bool later, int kv) {
  return ((int64_t)(2 * span + later) * a.batch.kv_heads + kv) * kFewRows;
}

// Blocks b0 .. b1 - 1 of sequence s at key-value head kv; `part`: its row among the parts, or
// negative where these are all of its blocks.
template <typename T, int D>
__device__ __forceinline__ void few_part(const Attention &a, int s, int kv, int b0, int b1,
                                         int64_t part, char *lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const PagedSequence seq = paged_sequence(a.batch, s, a.tokens);
  const int rows = seq.count * a.group;
  const int col = min(lane & 15, rows - 1), g = lane >> 4;
  const RowPlace at = row_place(a, seq, kv, col);
  u32x4 q[D / 32];
  const uint16_t *qr = a.q + (int64_t)at.token * a.q_token + (int64_t)at.head * a.q_head;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) q[i] = ldg16(qr + i * 32 + g * 8) ^ a.flip;

  FewKeys f;
  const int64_t head = (int64_t)(kv << a.batch.page_shift) * D;
  f.k = a.k_pages + head, f.v = a.v_pages + head;
  f.table = a.batch.table + s * a.batch.table_stride;
  f.page_stride = a.batch.page_stride, f.shift = a.batch.page_shift;
  f.pages = a.batch.pages, f.entries = a.batch.table_pages;
  const int last = min(b1 * (kBlockKeys / 16), (seq.length + 15) / 16);
  f.first = b0 * (kBlockKeys / 16) + wave, f.stride = kFewWaves;
  f.steps = last > f.first ? (last - f.first + kFewWaves - 1) / kFewWaves : 0;
  const int limit = min(seq.base + col / a.group + 1, seq.length);
  const int all_see = min(seq.base + 1, seq.length);  // keys that every row sees

  FewState<D> st;
  if (f.steps > 0) {
    few_pages(f, 0, lane);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) settle(q[i]);
    LDS char *ring = (LDS char *)lds + wave * few_ring<D>();
    constexpr int TILE = 16 * D * 2, STEPS = few_steps<D>();
    for (int j = 0; j < STEPS; ++j) {  // in this order: the waits count what was issued later
      few_load<D>(f, f.k, j, ring + 2 * j * TILE, lane);
      asm volatile("" ::: "memory");
      few_load<D>(f, f.v, j, ring + (2 * j + 1) * TILE, lane);
      asm volatile("" ::: "memory");
    }
    for (int i = 0; i < f.steps; ++i) {
      if (((i + STEPS) & 63) == 0) few_pages(f, i + STEPS, lane);  // that step is loaded next
      few_step<T, D>(ring, f, q, i, limit, all_see, a.scale2, st, lane);
    }
    wait_loads<0>();  // the last refills, before the ring is used otherwise
    if (__builtin_expect(st.odd, 0)) {
      for (int i = 0; i < f.steps; ++i) {
        const int key = (f.first + i * f.stride) * 16;
        if (key + 16 <= all_see) continue;
        for (int k = key; k < min(key + 16, limit); ++k) {
          const uint16_t *v = value_row<D>(a, s, head, k) + g * 4;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) st.o[j] += odd_parts<T>(v + j * 16);
        }
      }
    }
  }

  // The waves' sums, scaled to the largest of their maxima.
  __syncthreads();
  float *sums = reinterpret_cast<float *>(lds);  // [wave][row][D + 4]
  float *ml = sums + kFewWaves * kFewRows * (D + 4);  // [wave][row] maxima, then sums
  st.l = across32(across16(st.l, Add()), Add());
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    *reinterpret_cast<f32x4 *>(sums + (wave * kFewRows + (lane & 15)) * (D + 4) + i * 16 + g * 4) =
        st.o[i];
  if (lane < 16) {
    ml[wave * kFewRows + lane] = st.m;
    ml[(kFewWaves + wave) * kFewRows + lane] = st.l;
  }
  __syncthreads();
  for (int i = tid; i < rows * (D / 4); i += 256) {
    const int c = i / (D / 4), d = i % (D / 4) * 4;
    float m = ml[c], l = 0.0f;
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) m = fmaxf(m, ml[w * kFewRows + c]);
    f32x4 o = {};
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w) {
      const float k = decay(ml[w * kFewRows + c], m);
      l += ml[(kFewWaves + w) * kFewRows + c] * k;
      o += *reinterpret_cast<const f32x4 *>(sums + (w * kFewRows + c) * (D + 4) + d) * k;
    }
    if (part < 0) {
      const RowPlace to = row_place(a, seq, kv, c);
      write_row<T, D>(a, to, d, o * (l > 0.0f || l != l ? 1.0f / l : 0.0f), load_gate(a, to, d));
    } else {
      *reinterpret_cast<f32x4 *>(a.part + (part + c) * D + d) = o;
      if (d == 0) *reinterpret_cast<float2 *>(a.part_ml + (part + c) * 2) = float2{m, l};
    }
  }
  __syncthreads();  // before the ring is used again
}

template <typename T, int D>
__global__ __launch_bounds__(256, 1) void attention_few_kernel(Attention a) {
  // One array: with several, the compiler waits for all direct loads at each LDS read.
  __shared__ __attribute__((aligned(16))) char lds[few_lds<D>()];
  int64_t *scratch = reinterpret_cast<int64_t *>(lds);
  const int kv = blockIdx.x % a.batch.kv_heads, span = blockIdx.x / a.batch.kv_heads;
  Find at;
  const Spans sp = find_span(a, span, scratch, reinterpret_cast<Find *>(scratch + 8), at);
  if (at.s < 0) return;
  int64_t block = sp.start(span);
  const int64_t end = sp.start(span + 1);
  int s = __builtin_amdgcn_readfirstlane(at.s);
  int done = __builtin_amdgcn_readfirstlane((int)(block - at.first));  // blocks of s before
  bool later = false;
  for (; block < end && s < a.batch.sequences; ++s, done = 0) {
    const int all = __builtin_amdgcn_readfirstlane(few_blocks(a, s));
    const int take = __builtin_amdgcn_readfirstlane((int)min((int64_t)(all - done), end - block));
    if (take <= 0) continue;
    if (done == 0 && threadIdx.x == 0)  // where its parts are, for the kernel that joins them
      a.parts[s * a.batch.kv_heads + kv] = {span, later, sp.of(block + all - 1) - span + 1};
    few_part<T, D>(a, s, kv, done, done + take, take == all ? -1 : part_row(a, span, later, kv),
                   lds);
    block += take;
    later = true;
  }
}

// The sum of parts of a row: a thread's four channels, under the largest maximum so far.
struct PartSum {
  float m = -INFINITY, l = 0.0f;
  f32x4 o = {};
  __device__ __forceinline__ void add(float pm, float pl, f32x4 po) {
    const float n = fmaxf(m, pm), mine = decay(m, n), theirs = decay(pm, n);
    m = n;
    l = l * mine + pl * theirs;
    o = o * mine + po * theirs;
  }
  __device__ __forceinline__ float inverse() const { return l > 0.0f || l != l ? 1.0f / l : 0.0f; }
};

constexpr int kFewParts = 16;

// Rows of sequences whose keys attention_few_kernel split, by `ys` workgroups for a sequence's
// key-value head (`pair`).  Up to kFewParts parts: a thread takes four channels of a row, eight
// parts of it loaded at a time.  More: the workgroups share the rows and their channels, 64 at
// a time, the 16 groups of 16 threads the parts.
template <typename T, int D>
__device__ __forceinline__ void combine_few(const Attention &a, int pair, int y, int ys) {
  __shared__ __attribute__((aligned(16))) float sums[16][64];
  __shared__ float ms[16], ls[16];
  const int kv = pair % a.batch.kv_heads, s = pair / a.batch.kv_heads;
  const int tid = threadIdx.x, group = tid / 16;
  const Parts parts = a.parts[pair];
  const PagedSequence seq = paged_sequence(a.batch, s, a.tokens);
  if (!few_rows(seq, a.group) || parts.count < 2) return;
  const int rows = seq.count * a.group, n = parts.count;
  auto part = [&](int j, int c) {
    return part_row(a, parts.span + j, j == 0 && parts.later, kv) + c;
  };
  if (n <= kFewParts) {
    for (int u = y * 256 + tid; u < rows * (D / 4); u += ys * 256) {
      const int c = u / (D / 4), d = u % (D / 4) * 4;
      const RowPlace to = row_place(a, seq, kv, c);
      const uint2 gate = load_gate(a, to, d);
      PartSum sum;
      for (int j0 = 0; j0 < n; j0 += 8) {
        float2 ml[8];
        f32x4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int64_t row = part(min(j0 + j, n - 1), c);
          ml[j] = *reinterpret_cast<const float2 *>(a.part_ml + row * 2);
          v[j] = *reinterpret_cast<const f32x4 *>(a.part + row * D + d);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j0 + j < n) sum.add(ml[j].x, ml[j].y, v[j]);
      }
      write_row<T, D>(a, to, d, sum.o * sum.inverse(), gate);
    }
    return;
  }
  for (int u = y; u < rows * (D / 64); u += ys) {
    const int c = u / (D / 64), d = u % (D / 64) * 64 + tid % 16 * 4;
    const RowPlace to = row_place(a, seq, kv, c);
    const uint2 gate = load_gate(a, to, d);
    PartSum sum;
#pragma unroll 8
    for (int j = group; j < n; j += 16) {
      const int64_t row = part(j, c);
      const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + row * 2);
      sum.add(ml.x, ml.y, *reinterpret_cast<const f32x4 *>(a.part + row * D + d));
    }
    *reinterpret_cast<f32x4 *>(&sums[group][tid % 16 * 4]) = sum.o;
    if (tid % 16 == 0) ms[group] = sum.m, ls[group] = sum.l;
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int w = 1; w < 16; ++w)
        sum.add(ms[w], ls[w], *reinterpret_cast<const f32x4 *>(&sums[w][tid * 4]));
      write_row<T, D>(a, to, d, sum.o * sum.inverse(), gate);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ tiles
constexpr int kTileRows = 128;  // rows of a tile, 32 a wave

// Key groups of a workgroup: as many waves more take other keys of a tile for the same rows,
// and their sums are joined in LDS at the end.
template <int D>
struct TileForm {
  static constexpr int kGroups = D == 256 ? 2 : 1;
  static constexpr int kWaves = 4 * kGroups, kKeys = 32 * kGroups;
};

// Tiles of the rows of sequence s, unless the few-row kernel takes them.
__device__ __forceinline__ int tile_count(const Attention &a, int s) {
  if (s >= a.batch.sequences) return 0;
  const PagedSequence q = paged_sequence(a.batch, s, a.tokens);
  if (a.few && few_rows(q, a.group)) return 0;
  return (int)(((int64_t)q.count * a.group + kTileRows - 1) / kTileRows);
}

// Keys that the last row of a sequence's tile sees, the most of its rows.
__device__ __forceinline__ int tile_keys(const PagedSequence &q, int group, int tile) {
  const int last = min((int64_t)(tile + 1) * kTileRows, (int64_t)q.count * group) - 1;
  return max(min(q.base + last / group + 1, q.length), 0);
}

// Keys of n tiles of sequence s together (their mean is that of the first and the last).
__device__ __forceinline__ int64_t all_keys(const Attention &a, int s, int n) {
  if (n == 0) return 0;
  const PagedSequence q = paged_sequence(a.batch, s, a.tokens);
  return ((int64_t)tile_keys(q, a.group, 0) + tile_keys(q, a.group, n - 1)) * n / 2;
}

struct TilePlace {
  int s, tile;   // s < 0: none
  // where tiles are split each in its own way: all tiles of the call, and their keys
  int tiles;
  int64_t keys;
};

// Parts of a tile that sees `keys` keys, where sequences differ: about equal parts, as many as
// the tiles, which take one or more each, leave of so many rounds of workgroups that they fill
// two thirds at most; none below 256 keys.  Against as many parts for every tile, 12 sequences of
// up to 700 new tokens took 52 us instead of 61 (heads of 128) and 61 instead of 77 (256), 24 of
// 8 to 24 tokens 46 instead of 55; parts of 128 or 512 keys and fewer or more rounds took up to
// 30 % more in one case or another.
__device__ __forceinline__ int tile_parts(const Attention &a, const TilePlace &place, int keys) {
  const int rounds = (int)((float)place.tiles * 1.5f / (float)a.room) + 1;
  const float all = (float)max(place.keys, (int64_t)1);
  const float n = (float)keys * (float)(rounds * a.room - place.tiles) / all + 0.5f;
  return max(min(min((int)fminf(n, 65536.0f), a.splits), keys / 256), 1);
}

// The index-th tile; the tile with the most keys of a sequence comes first.
// All THREADS threads; scratch (a word and a long word a wave) and found are free again
// afterwards.
template <int THREADS>
__device__ TilePlace find_tile(const Attention &a, int index, int *scratch, int64_t *sums,
                               TilePlace *found) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool split = a.room > 0;
  if (a.batch.sequences == 1) {
    const int n = tile_count(a, 0);
    return {index < n ? 0 : -1, n - 1 - index, 0, 0};
  }
  auto scan = [&](int &sum, int64_t &keys) {  // counts up to the lane's, keys of all lanes
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o, 64);
      if (lane >= o) sum += v;
    }
    if (split)
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) keys += __shfl_xor(keys, o, 64);
  };
  if (a.batch.sequences <= 64) {  // each wave for itself
    const int n = tile_count(a, lane);
    int sum = n;
    int64_t keys = split ? all_keys(a, lane, n) : 0;
    scan(sum, keys);
    const uint64_t hit = __ballot(index >= sum - n && index < sum);
    if (!hit) return {-1, 0, 0, 0};
    const int at = __builtin_ctzll(hit);
    return {at, __shfl(sum, at, 64) - 1 - index, __shfl(sum, 63, 64), keys};
  }
  if (tid == 0) found->s = -1;
  int base = 0;
  int64_t all = 0;
  for (int c = 0; c < a.batch.sequences; c += THREADS) {
    const int n = tile_count(a, c + tid);
    int sum = n;
    int64_t keys = split ? all_keys(a, c + tid, n) : 0;
    scan(sum, keys);
    __syncthreads();
    if (lane == 63) scratch[wave] = sum, sums[wave] = keys;
    __syncthreads();
    int before = base;
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) before += scratch[w];
      base += scratch[w], all += sums[w];
    }
    before += sum - n;
    if (index >= before && index < before + n) *found = {c + tid, n - 1 - (index - before), 0, 0};
    if (base > index && !split) break;  // the same for every thread
  }
  __syncthreads();
  TilePlace got = *found;
  got.tiles = base, got.keys = all;
  __syncthreads();
  return got;
}

template <int D>
struct TileState {
  float m = -INFINITY, l = 0.0f;  // of column lane & 31; l: this lane's keys only
  f32x16 o[D / 32] = {};          // o[i][4 b + r]: channel 32 i + 8 b + 4 (lane >> 5) + r
  bool odd = false;               // infinities or NaN were left out
};

// Where a wave finds the keys of a tile: the pages of 64 steps of 16 keys from `from` on, one
// a lane.
struct TilePages {
  const int32_t *table;
  int64_t page_stride;
  const uint16_t *k, *v;  // of the key-value head, in page 0
  int shift, pages, entries;
  int from, page_of;
};

__device__ __forceinline__ void tile_pages(TilePages &f, int key, int lane) {
  f.from = key;
  const int i = min((key + lane * 16) >> f.shift, f.entries - 1);
  f.page_of = clamp_index32(f.table[i], f.pages);
  settle(f.page_of);
}

// Loads a tile of keys and values from `key` on into LDS: ROWS rows of each a wave.
template <int D, int ROWS>
__device__ __forceinline__ void tile_load(TilePages &f, int key, LDS char *kt, LDS char *vt,
                                          int wave, int lane) {
  if (key - f.from >= 1024) tile_pages(f, key, lane);
#pragma unroll
  for (int r = 0; r < ROWS; r += 16) {  // of one page each
    constexpr int N = ROWS < 16 ? ROWS : 16;
    const int row = wave * ROWS + r, k = key + row, to = row * D * 2;
    const int page = __builtin_amdgcn_readlane(f.page_of, (k - f.from) >> 4);
    const int64_t at = page * f.page_stride + (int64_t)(k & ((1 << f.shift) - 1)) * D;
    load_rows<D, N>(f.k + at, row, kt + to, lane);
    load_rows<D, N, kQuads>(f.v + at, row, vt + to, lane);
  }
}

// Operands that are read from LDS before the product that needs the first of them.  Left to its
// own order, the compiler waits for each operand right before its product: 9 % more time with
// heads of 256 (2048 tokens behind 8192 keys: 374 us instead of 337), 3 % with 128.
constexpr int kAheadReads = 4;

// Operand of 16 keys from row `ks` of the tile, channels 32 i ..
template <int D>
__device__ __forceinline__ u32x4 tile_operand(const LDS char *vt, int base, int i, int ks) {
  const u32x2 lo = read_transposed<D, kQuads>(vt, base, ks, i * 32);
  const u32x2 hi = read_transposed<D, kQuads>(vt, base, ks + 8, i * 32);
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// Adds the weighted values of 32 keys; MIXED: some row does not see all of them.
template <typename T, int D, bool MIXED>
__device__ __forceinline__ void tile_values(const LDS char *vt, const u32x4 (&p)[2],
                                            TileState<D> &st, int lane) {
  const int base = opaque(transpose_base<D, kQuads>((lane >> 5) * 4, ((lane >> 4) & 1) * 16, lane));
  if constexpr (MIXED) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        u32x4 v = tile_operand<D>(vt, base, i, ks * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = Pair<T>::finite(v[j], any);
        st.o[i] = mfma32(T{}, v, p[ks], st.o[i]);
      }
    st.odd |= __any(any != 0);
    return;
  }
  __builtin_amdgcn_s_setprio(1);
  u32x4 v[kAheadReads];
#pragma unroll
  for (int u = 0; u < kAheadReads; ++u) v[u] = tile_operand<D>(vt, base, u / 2, u % 2 * 16);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int u = 0; u < D / 16; ++u) {
    st.o[u / 2] = mfma32(T{}, v[u % kAheadReads], p[u % 2], st.o[u / 2]);
    const int n = u + kAheadReads;
    if (n < D / 16) v[u % kAheadReads] = tile_operand<D>(vt, base, n / 2, n % 2 * 16);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
}

// 32 keys of a tile for a wave's 32 rows.  MIXED: some row does not see all of them.
// The wave's priority is raised while it feeds the matrix cores, so that the other wave of
// its SIMD does its softmax beside them.
template <typename T, int D, bool MIXED>
__device__ __forceinline__ void tile_step(const LDS char *kt, const LDS char *vt,
                                          const u32x4 (&q)[D / 16], int key, int limit,
                                          float scale2, TileState<D> &st, int lane) {
  const int h = lane >> 5, r = lane & 31;
  const int base = opaque(r * (D * 2) + ((h ^ swizzle<D>(r)) << 4));
  f32x16 x = {};
  __builtin_amdgcn_s_setprio(1);
  auto read = [&](int i) { return *(const LDS u32x4 *)(kt + swizzled<D, kRows>(base, 0, i * 2)); };
  u32x4 k[kAheadReads];
#pragma unroll
  for (int i = 0; i < kAheadReads; ++i) k[i] = read(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    x = mfma32(T{}, k[i % kAheadReads], q[i], x);
    if (i + kAheadReads < D / 16) k[i % kAheadReads] = read(i + kAheadReads);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
  if constexpr (MIXED) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (key + 8 * (i / 4) + 4 * h + i % 4 >= limit) x[i] = -INFINITY;
  }
  float mx = x[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
  mx = __builtin_fmaf(across32(mx, Max()), scale2, -kLift<T>);
  if (__any(mx > st.m + kSlack)) {
    const float n = fmaxf(st.m, mx), keep = decay(st.m, n);
    st.m = n;
    st.l *= keep;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) st.o[i] *= keep;
  }
  const float at = st.m == -INFINITY ? 0.0f : st.m;
  u32x4 p[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float e0 = exp2_hw(__builtin_fmaf(x[2 * i], scale2, -at));
    const float e1 = exp2_hw(__builtin_fmaf(x[2 * i + 1], scale2, -at));
    st.l += e0 + e1;
    p[i / 4][i % 4] = T::pack2(e0, e1);
  }
  tile_values<T, D, MIXED>(vt, p, st, lane);
}

// The waves' sums on their way out, half of the channels at a time: rows of D / 2 channels
// and a pad of four, then each row's maximum and sum.
template <int D>
constexpr int tile_pitch() { return D / 2 + 4; }
template <int D>
constexpr int tile_lds() {
  using F = TileForm<D>;
  constexpr int ring = 4 * F::kKeys * D * 2, out = F::kWaves * 32 * (tile_pitch<D>() + 2) * 4;
  return out > ring ? out : ring;
}

template <typename T, int D>
__global__ __launch_bounds__(TileForm<D>::kWaves * 64, 2) void attention_tile_kernel(Attention a) {
  constexpr int WAVES = TileForm<D>::kWaves, KEYS = TileForm<D>::kKeys, ROWS = KEYS / WAVES;
  constexpr int GROUPS = TileForm<D>::kGroups, TILE = KEYS * D * 2;
  static_assert(GROUPS == 1 || GROUPS == 2, "two groups are joined");
  // One array: with several, the compiler waits for all direct loads at each LDS read.
  __shared__ __attribute__((aligned(16))) char lds[tile_lds<D>()];
  int *scratch = reinterpret_cast<int *>(lds);
  int64_t *key_sums = reinterpret_cast<int64_t *>(scratch + 8);
  TilePlace *found = reinterpret_cast<TilePlace *>(key_sums + 8);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int set = wave & 3, group = wave >> 2;
  const int kv = blockIdx.x % a.batch.kv_heads, split = blockIdx.y;
  const TilePlace place =
      find_tile<WAVES * 64>(a, blockIdx.x / a.batch.kv_heads, scratch, key_sums, found);
  const int s = __builtin_amdgcn_readfirstlane(place.s);
  if (s < 0) return;
  const PagedSequence seq = paged_sequence(a.batch, s, a.tokens);
  const int tile = __builtin_amdgcn_readfirstlane(place.tile);
  const int rows = seq.count * a.group, c0 = tile * kTileRows;
  const int c = c0 + set * 32 + (lane & 31);
  const bool idle = c0 + set * 32 >= rows;
  const RowPlace at = row_place(a, seq, kv, min(c, rows - 1));
  const int limit = min(seq.base + min(c, rows - 1) / a.group + 1, seq.length);
  const int all_see = min(seq.base + c0 / a.group + 1, seq.length);  // seen by every row
  // keys that the tile's last row sees, and this part of them
  const int keys = tile_keys(seq, a.group, tile), tiles = (keys + KEYS - 1) / KEYS;
  const int splits = __builtin_amdgcn_readfirstlane(a.room ? tile_parts(a, place, keys) : a.splits);
  if (split >= splits) return;
  const int key0 = (int)((int64_t)tiles * split / splits) * KEYS;
  const int key1 = min((int)((int64_t)tiles * (split + 1) / splits) * KEYS, keys);

  u32x4 q[D / 16];
  const uint16_t *qr = a.q + (int64_t)at.token * a.q_token + (int64_t)at.head * a.q_head + (lane >> 5) * 8;
  TileState<D> st;
  LDS char *base = (LDS char *)lds;
  const int64_t head = (int64_t)(kv << a.batch.page_shift) * D;
  if (key0 < key1) {
    TilePages f;
    f.table = a.batch.table + s * a.batch.table_stride, f.page_stride = a.batch.page_stride;
    f.k = a.k_pages + head, f.v = a.v_pages + head, f.shift = a.batch.page_shift;
    f.pages = a.batch.pages, f.entries = a.batch.table_pages;
    tile_pages(f, key0, lane);
    tile_load<D, ROWS>(f, key0, base, base + TILE, wave, lane);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) q[i] = ldg16(qr + i * 16) ^ a.flip;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) settle(q[i]);
    wait_loads<0>();
    __syncthreads();
    // A tile, the next one's loads started before it into the other half.
    int key = key0, half = 0;
    const int whole = min(key1, all_see), own = group * 32;
    for (; key + KEYS <= whole; key += KEYS, half ^= 1) {
      LDS char *cur = base + half * 2 * TILE, *next = base + (half ^ 1) * 2 * TILE;
      if (key + KEYS < key1) tile_load<D, ROWS>(f, key + KEYS, next, next + TILE, wave, lane);
      if (!idle)
        tile_step<T, D, false>(cur + own * D * 2, cur + TILE + own * D * 2, q, key + own, limit,
                               a.scale2, st, lane);
      wait_loads<0>();
      __syncthreads();
    }
    for (; key < key1; key += KEYS, half ^= 1) {
      LDS char *cur = base + half * 2 * TILE, *next = base + (half ^ 1) * 2 * TILE;
      if (key + KEYS < key1) tile_load<D, ROWS>(f, key + KEYS, next, next + TILE, wave, lane);
      if (!idle)
        tile_step<T, D, true>(cur + own * D * 2, cur + TILE + own * D * 2, q, key + own, limit,
                              a.scale2, st, lane);
      wait_loads<0>();
      __syncthreads();
    }
    if (__builtin_expect(st.odd, 0)) {
      for (int k = key0 + max(all_see - key0, 0) / KEYS * KEYS; k < min(key1, limit); ++k) {
        if (((k - key0) / 32) % GROUPS != group) continue;
        const uint16_t *v = value_row<D>(a, s, head, k) + (lane >> 5) * 4;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const f32x4 x = odd_parts<T>(v + i * 32 + b * 8);
#pragma unroll
            for (int j = 0; j < 4; ++j) st.o[i][4 * b + j] += x[j];
          }
      }
    }
  }

  // Through LDS, which every wave has left: the last barrier above, or no key at all.  The
  // key groups' sums are joined on the way, and rows are written whole.
  constexpr int PITCH = tile_pitch<D>(), C = D / 2;
  float *sums = reinterpret_cast<float *>(lds), *ml = sums + WAVES * 32 * PITCH;
  const float l = across32(st.l, Add());
  if (lane < 32) {
    ml[(wave * 32 + lane) * 2] = st.m;
    ml[(wave * 32 + lane) * 2 + 1] = l;
  }
  __syncthreads();
  if (threadIdx.x < kTileRows) {  // what each group's sum of a row counts for
    PartSum sum;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const float *p = ml + (g * kTileRows + threadIdx.x) * 2;
      sum.add(p[0], p[1], f32x4{});
    }
    const float inv = splits == 1 ? sum.inverse() : 1.0f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      float *p = ml + (g * kTileRows + threadIdx.x) * 2;
      p[0] = decay(p[0], sum.m) * inv;
    }
    if (a.splits > 1 && c0 + threadIdx.x < rows) {
      const RowPlace to = row_place(a, seq, kv, c0 + threadIdx.x);
      const int64_t row = (int64_t)to.token * a.q_heads + to.head;
      if (a.room && split == 0) a.row_parts[row] = splits;
      if (splits > 1)
        *reinterpret_cast<float2 *>(a.tile_ml + ((int64_t)split * a.tokens * a.q_heads + row) * 2) =
            float2{sum.m, sum.l};
    }
  }
  // A thread's units of four channels lie STEP rows apart; four at a time, their gates first.
  // Little code, as it runs once: unrolled, it took longer to fetch than to run.
  constexpr int STEP = WAVES * 64 / (C / 4), BATCH = 4;
  const int first = threadIdx.x / (C / 4), d = threadIdx.x % (C / 4) * 4;
  const int live = min(rows - c0, kTileRows), step_t = STEP / a.group, step_h = STEP % a.group;
  const int t0 = (c0 + first) / a.group, h0 = (c0 + first) % a.group;
  auto put = [&](const f32x16 &o, int i) {
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *reinterpret_cast<f32x4 *>(sums + (wave * 32 + (lane & 31)) * PITCH + i * 32 + b * 8 +
                                 (lane >> 5) * 4) =
          f32x4{o[4 * b], o[4 * b + 1], o[4 * b + 2], o[4 * b + 3]};
  };
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    if (side == 0) {
#pragma unroll
      for (int i = 0; i < D / 64; ++i) put(st.o[i], i);
    } else {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < D / 64; ++i) put(st.o[D / 64 + i], i);
    }
    __syncthreads();
    int t = t0, h = h0;
#pragma unroll 1
    for (int r0 = first; r0 < live; r0 += BATCH * STEP) {
      uint2 gate[BATCH];
      RowPlace to[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        to[i] = {seq.first + min(t, seq.count - 1), kv * a.group + h};
        if (splits == 1) gate[i] = load_gate(a, to[i], side * C + d);
        t += step_t, h += step_h;
        if (h >= a.group) h -= a.group, ++t;
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int r = r0 + i * STEP;
        if (r >= live) break;
        f32x4 o = *reinterpret_cast<const f32x4 *>(sums + r * PITCH + d) * ml[r * 2];
        if constexpr (GROUPS == 2) {
          const int w = kTileRows + r;
          o += *reinterpret_cast<const f32x4 *>(sums + w * PITCH + d) * ml[w * 2];
        }
        if (splits == 1) {
          write_row<T, D>(a, to[i], side * C + d, o, gate[i]);
        } else {
          const int64_t row = ((int64_t)split * a.tokens + to[i].token) * a.q_heads + to[i].head;
          *reinterpret_cast<f32x4 *>(a.tile_part + row * D + side * C + d) = o;
        }
      }
    }
  }
}

// Rows of sequences in tiles, where their keys were split: D / 4 threads a row, `chunks`
// workgroups a token.
template <typename T, int D>
__device__ __forceinline__ void combine_tile(const Attention &a, int block, int chunks) {
  const int t = block / chunks, lane = threadIdx.x & 63;
  const int i = block % chunks * 256 + threadIdx.x;
  const int head = i / (D / 4), d = i % (D / 4) * 4;
  int s = -1;  // the token's sequence: a lane looks at one of 64
  for (int c = 0; c < a.batch.sequences && s < 0; c += 64) {
    const int k = c + lane;
    const uint64_t hit = __ballot(k < a.batch.sequences && a.batch.starts[min(k, a.batch.sequences - 1)] <= t &&
                                  t < a.batch.starts[min(k, a.batch.sequences - 1) + 1]);
    if (hit) s = c + __builtin_ctzll(hit);
  }
  if (s < 0 || head >= a.q_heads) return;
  const PagedSequence seq = paged_sequence(a.batch, s, a.tokens);
  if (t < seq.first || t >= seq.first + seq.count || (a.few && few_rows(seq, a.group))) return;
  const int64_t rows = (int64_t)a.tokens * a.q_heads, row = (int64_t)t * a.q_heads + head;
  const int parts = a.room ? min(a.row_parts[row], a.splits) : a.splits;
  if (parts < 2) return;  // written by its tile
  const uint2 gate = load_gate(a, {t, head}, d);
  PartSum sum;
  for (int j0 = 0; j0 < parts; j0 += 4) {
    float2 ml[4];
    f32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = row + min(j0 + j, parts - 1) * rows;
      ml[j] = *reinterpret_cast<const float2 *>(a.tile_ml + r * 2);
      v[j] = *reinterpret_cast<const f32x4 *>(a.tile_part + r * D + d);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j0 + j < parts) sum.add(ml[j].x, ml[j].y, v[j]);
  }
  write_row<T, D>(a, {t, head}, d, sum.o * sum.inverse(), gate);
}

// Joins the parts of both kernels in one launch (one for each took 2 us longer where a call
// has both): `ys` workgroups for each of the few rows' pairs, then those of the tiles.  The
// pairs' first workgroups come first, as in many pairs only those have work.
template <typename T, int D>
__global__ __launch_bounds__(256) void attention_combine_kernel(Attention a, int pairs, int ys, int chunks) {
  const int block = blockIdx.x;
  if (block < pairs * ys)
    combine_few<T, D>(a, block % pairs, block / pairs, ys);
  else
    combine_tile<T, D>(a, block - pairs * ys, chunks);
}

// ------------------------------------------------------------------ host side
// What a call launches, by its sizes alone.
struct AttentionPlan {
  bool few, tile;
  int64_t shares, few_grid;          // few: parts per key-value head, workgroups
  int64_t tiles, splits, room;       // tile: tiles at most, parts of each, see Attention
  int64_t few_rows, tile_rows, parts, row_parts;  // rows of partial sums, Parts, rows' parts
};

AttentionPlan attention_plan(int64_t tokens, int64_t sequences, int64_t q_heads, int64_t kv_heads,
                             int64_t head_dim, int64_t max_new, int64_t max_keys) {
  AttentionPlan p = {};
  const int64_t group = q_heads / kv_heads;
  max_new = max_new < tokens ? max_new : tokens;
  p.tile = max_new * group > kFewRows;
  p.few = group <= kFewRows && !(p.tile && sequences == 1);  // one sequence: one of them
  if (p.few) {
    const int64_t all = head_dim == 64 ? 768 : 512;  // workgroups that run at a time
    p.shares = all / kv_heads > 1 ? all / kv_heads : 1;
    p.few_grid = p.shares * kv_heads;
    p.few_rows = 2 * p.shares * kv_heads * kFewRows;
    p.parts = sequences * kv_heads;
  }
  if (p.tile) {
    const int64_t some = sequences < tokens ? sequences : tokens;
    p.tiles = tokens * group / kTileRows + some;
    // One sequence's tiles have nearly the same keys: as many parts for each as keep the
    // workgroups within two rounds.  Others differ: see tile_parts.
    const int64_t round = (head_dim == 256 ? 256 : 512), pairs = p.tiles * kv_heads;
    int64_t n = 2 * round / pairs, most = max_keys / 256;
    if (sequences > 1 && n > 0) n = 4 * round / pairs + 1;
    p.splits = n < most ? n : most;
    if (p.splits < 1) p.splits = 1;
    if (p.splits > 1) {
      p.tile_rows = p.splits * tokens * q_heads;
      if (sequences > 1) {
        p.room = round / 2 / kv_heads > 1 ? round / 2 / kv_heads : 1;
        p.row_parts = tokens * q_heads;
      }
    }
  }
  return p;
}

int64_t attention_bytes(const AttentionPlan &p, int64_t head_dim) {
  return (p.few_rows + p.tile_rows) * (head_dim + 2) * 4 + p.row_parts * 4 +
         (p.parts * sizeof(Parts) + 15) / 16 * 16;
}

template <typename T, int D>
int launch_attention(const AttentionPlan &p, Attention a, float *workspace, hipStream_t st) {
  a.few = p.few;
  a.part = workspace, a.part_ml = workspace + p.few_rows * D;
  a.tile_part = workspace + p.few_rows * (D + 2), a.tile_ml = a.tile_part + p.tile_rows * D;
  a.parts = reinterpret_cast<Parts *>(a.tile_ml + p.tile_rows * 2);
  a.row_parts = reinterpret_cast<int *>(a.parts + p.parts);
  a.shares = (int)p.shares, a.splits = (int)p.splits, a.room = (int)p.room;
  int64_t ys = 0, tile = 0;  // workgroups that join parts: ys for each of p.parts, and tile
  if (p.few) {
    attention_few_kernel<T, D><<<(unsigned)p.few_grid, 256, 0, st>>>(a);
    if (const int rc = check_launch("attention_few_kernel")) return rc;
    // Where there are few sequences, their rows and channels fill the chip.
    const int64_t units = kFewRows / a.group * a.group * (D / 64), some = 4096 / p.parts;
    ys = some < 1 ? 1 : some < units ? some : units;
  }
  const int chunks = (a.q_heads * (D / 4) + 255) / 256;
  if (p.tile) {
    const dim3 grid((unsigned)(p.tiles * a.batch.kv_heads), (unsigned)p.splits);
    attention_tile_kernel<T, D><<<grid, TileForm<D>::kWaves * 64, 0, st>>>(a);
    if (const int rc = check_launch("attention_tile_kernel")) return rc;
    if (p.splits > 1) tile = (int64_t)a.tokens * chunks;
  }
  const int64_t all = p.parts * ys + tile;
  if (all == 0) return LM_OK;
  attention_combine_kernel<T, D><<<(unsigned)all, 256, 0, st>>>(a, (int)p.parts, (int)ys, chunks);
  return check_launch("attention_combine_kernel");
}

template <typename T>
int launch_attention(const AttentionPlan &p, const Attention &a, float *workspace, int head_dim,
                     hipStream_t st) {
  return head_dim == 256   ? launch_attention<T, 256>(p, a, workspace, st)
         : head_dim == 128 ? launch_attention<T, 128>(p, a, workspace, st)
                           : launch_attention<T, 64>(p, a, workspace, st);
}

}  // namespace
}  // namespace lm

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
  if (const int rc = paged_check(pages, page_stride, kv_heads, page_size, head_dim, starts, lengths,
                                 table, table_stride, table_pages, sequences, tokens, dtype))
    return rc;
  LM_REQUIRE(q_heads >= 1 && q_heads <= 16384 && q_heads % kv_heads == 0, LM_EINVAL,
             "query heads must be a multiple of key-value heads");
  LM_REQUIRE(max_new >= 0, LM_EINVAL, "invalid number of new tokens");
  const float scale2 = fabsf(scale) * 1.4426950408889634f;
  LM_REQUIRE(std::isfinite(scale2), LM_EINVAL, "the scale must be finite");
  if (tokens == 0 || sequences == 0) return LM_OK;
  LM_REQUIRE(tokens * q_heads < (1LL << 31), LM_EINVAL, "too many rows");
  LM_REQUIRE(q && k_pages && v_pages && out, LM_EINVAL, "null pointer");
  LM_REQUIRE(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out) &&
                 q_token_stride % 8 == 0 && q_head_stride % 8 == 0 && q_token_stride >= 0 &&
                 q_head_stride >= 0,
             LM_EINVAL, "head rows must be 16-byte aligned");
  LM_REQUIRE(!gate || (aligned16(gate) && gate_token_stride % 8 == 0 && gate_head_stride % 8 == 0 &&
                       gate_token_stride >= 0 && gate_head_stride >= 0),
             LM_EINVAL, "head rows must be 16-byte aligned");
  const AttentionPlan plan = attention_plan(tokens, sequences, q_heads, kv_heads, head_dim, max_new,
                                            table_pages * page_size);
  // threads of the largest launches, below 2^32
  LM_REQUIRE(sequences * kv_heads < (1LL << 24) && plan.tiles * kv_heads < (1LL << 23), LM_EINVAL,
             "too many rows");
  const int64_t need = attention_bytes(plan, head_dim);
  LM_REQUIRE(need == 0 || (workspace && aligned16(workspace)), LM_EINVAL,
             "attention needs a 16-byte aligned workspace");
  LM_REQUIRE(workspace_bytes >= need, LM_ENOMEM, "the workspace is too small");
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
  // A scale of 0 as one too small to matter, so that a masked -inf stays one under it.
  a.scale2 = fmaxf(scale2, 1e-30f);
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  float *ws = static_cast<float *>(workspace);
  return dtype == LM_BF16
             ? launch_attention<BF16>(plan, a, ws, (int)head_dim, as_stream(stream))
             : launch_attention<FP16>(plan, a, ws, (int)head_dim, as_stream(stream));
}
