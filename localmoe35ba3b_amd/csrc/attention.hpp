// Attention of each sequence's new tokens over its paged cache (gfx950), which holds values of
// the rows' type (attention.hip) or of 8 bits (attention_e4m3.hip).
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
//                         behind 8192 keys: 293 to 306 us on the same inputs, 320
//                         on others each time, 966 to 1054 TFLOP/s (1372 for a
//                         large library product); without a history 64 to 75 us.
//  attention_both_kernel  the two in one launch, for calls that may have both (not with
//                         heads of 256 in 16 bits).
//  attention_combine_kernel  joins the parts of split keys, 3 to 10 us: the partial
//                         sums are fp32, written and read once.
//
// A cache of 8 bits, e4m3 with a power of two for each 16 positions of a head, goes the
// same way into LDS.  The values are multiplied by their scale as they become operands,
// four significant bits that the rows' type holds exactly, so all else is as above and
// a result is as far off.  A lane's 16 bytes of a key are the operands of two products
// (the queries' channels follow), and V^T comes from the 8-bit transpose read, eight
// keys of one channel a lane, so steps of few rows have 32 keys.  The conversions are 64
// instructions a wave and 32 keys of 256 channels, for K as for V, beside 32 products:
// the tiles of 256 channels take 1 to 5 % longer than with 16 bits, while the reads from
// LDS are half.  Two products' conversions made ahead gained 1 %.  A page's scales are
// looked up with it, 64 blocks a wave at a time, as two exponents in a lane's register.
// Times as above: 262144 keys 49 us (5.5 TB/s), 64 sequences 49 us (4.9 TB/s; of both
// some 6 us are the chain from lengths to pages to rows, before which nothing is under
// way), 2048 tokens behind 8192 keys 298 to 316 us.
#pragma once

#include <cmath>
#include <type_traits>
#include <utility>

#include "paged.hpp"

namespace lm {
namespace {

#define LDS __attribute__((address_space(3)))
#define GLB __attribute__((address_space(1)))

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

// What a cache holds: values of the rows' type T, or 8 bits with a scale (a power of two) for each
// kScaleKeys positions of a head and side.
template <typename C>
struct Cache {
  using Elem = uint16_t;
  static constexpr int kBytes = 2;      // of a value
  static constexpr int kFewKeys = 16;   // keys of a step of few rows
  static constexpr int kTileSteps = 1;  // steps of 32 keys that a wave takes of a tile
  static constexpr bool kScaled = false;
};
template <>
struct Cache<E4M3> {
  using Elem = uint8_t;
  static constexpr int kBytes = 1, kFewKeys = 32, kTileSteps = 2;
  static constexpr bool kScaled = true;
};

// The parts of a sequence at a key-value head: their first span, its place there, their count.
struct Parts {
  int span, later, count;
};

struct Attention {
  const uint16_t *q, *gate;  // gate: null or a row for each row of q
  int64_t q_token, q_head, gate_token, gate_head;  // strides, elements
  const void *k_pages, *v_pages;
  const float *scales;   // of 8 bits: [pages][kv_heads][2: keys, values][page_size / kScaleKeys]
  int64_t scale_stride;  // between pages, elements
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
// rows that one LDS read touches use different banks (rows of B bytes, the banks repeat every
// 256).  kRows: reads of one or two pieces of 16 rows; kQuads: of four pieces of 4 rows
// (the transpose reads of 32 channels; with kRows they took 4 times as long).  Of 8 bits a value:
// kOctets, two pieces of rows 0 .. 3 and 8 .. 11 of 16 (or the other eight); kHalves, one piece of
// rows 0 .. 7 and 16 .. 23 of 32 (or the others).  Linear over disjoint bits of r: a read's lane
// part is formed once, its constant part is one exclusive or.
enum Swizzle { kRows, kQuads, kOctets, kHalves };
template <int B, Swizzle S = kRows>
__device__ __forceinline__ constexpr int swizzle(int r) {
  if (S == kRows) return B == 64 ? (r >> 2) & 3 : B == 128 ? (r >> 1) & 7 : r & 15;
  if (S == kQuads) return B == 128 ? (r & 2) << 1 : (r & 3) << 2;
  if (S == kOctets)
    return B == 64 ? (r >> 2) & 2 : B == 128 ? (r & 2) | ((r >> 1) & 4) : (r & 3) << 1 | (r & 8);
  return B == 64    ? ((r >> 2) & 1) | ((r >> 3) & 2)
         : B == 128 ? ((r >> 1) & 3) | ((r >> 2) & 4)
                    : (r & 7) | ((r >> 1) & 8);
}

// Cache policy of loads that are not read again (non-temporal): 262144 keys of one sequence
// in 88 us instead of 96; the tiles, which other workgroups read too, take 10 % longer with it.
constexpr int kStream = 2;

// ROWS rows of a page, from `src` (row `row0` of the tile), into LDS: wave-wide loads of
// 1 KB, lane-linear in LDS, so the swizzle permutes the source.  Rows behind a sequence's
// end are loaded as they are (their page holds them) and masked later.  An instruction's
// offset counts for both addresses, so four share a pair of them.
template <int B, int PER, Swizzle S, int POLICY, int... I>
__device__ __forceinline__ void load_4k(const GLB char *from, uint32_t off, int row0, LDS char *to,
                                        std::integer_sequence<int, I...>) {
  (__builtin_amdgcn_global_load_lds(
       (const GLB void *)(from + (off ^ (swizzle<B, S>(row0 + I * PER) << 4))), (LDS void *)to, 16,
       I * 1024, POLICY),
   ...);
}
template <int B, int ROWS, Swizzle S = kRows, int POLICY = 0>
__device__ __forceinline__ void load_rows(const void *src, int row0, LDS char *to, int lane) {
  constexpr int PIECES = B / 16, PER = 64 / PIECES, LOADS = ROWS / PER, GROUP = LOADS < 4 ? LOADS : 4;
  static_assert(ROWS % PER == 0 && LOADS % GROUP == 0, "whole loads of 1 KB");
  const int own = lane / PIECES;
  const uint32_t off = own * B + (((lane % PIECES) ^ swizzle<B, S>(own)) << 4);
#pragma unroll
  for (int i = 0; i < LOADS / GROUP; ++i)
    load_4k<B, PER, S, POLICY>((const GLB char *)src + i * 4096, off, row0 + i * 4 * PER,
                               to + i * 4096, std::make_integer_sequence<int, GROUP>{});
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
template <int B, Swizzle S>
__device__ __forceinline__ int transpose_base(int row, int d, int lane) {
  const int r = row + (lane & 15) / 4;
  return r * B + (((d / 8 + (lane & 3) / 2) ^ swizzle<B, S>(r)) << 4) + (lane & 1) * 8;
}
// The address of piece `ch` (constant) of row `row` (constant) past a lane's base, in which
// the piece's low four bits were swizzled.
template <int B, Swizzle S>
__device__ __forceinline__ int swizzled(int base, int row, int ch) {
  return (base ^ (((ch & 15) ^ swizzle<B, S>(row)) << 4)) + (ch & 16) * 16 + row * B;
}
template <int B, Swizzle S>
__device__ __forceinline__ u32x2 read_transposed(const LDS char *tile, int base, int row, int d) {
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                 (LDS s16x4 *)(tile + swizzled<B, S>(base, row, d / 8))));
}

// Of 8 bits a value, eight keys of one channel: lane i of each 16 lanes gets channel i of a piece's
// 16 of rows row .. row + 3 and row + JUMP .. row + JUMP + 3, in that order.
template <int B, Swizzle S, int JUMP>
__device__ __forceinline__ int transpose8_base(int row, int piece, int lane) {
  const int i = (lane & 15) / 2, r = row + (i & 3) + (i >> 2) * JUMP;
  return r * B + ((piece ^ swizzle<B, S>(r)) << 4) + (lane & 1) * 8;
}
template <int B, Swizzle S>
__device__ __forceinline__ u32x2 read_transposed8b(const LDS char *tile, int base, int row,
                                                   int piece) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                       (LDS i32x2 *)(tile + swizzled<B, S>(base, row, piece))));
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
__device__ __forceinline__ void read_transposed8x8(u32x2 (&v)[8], const LDS char *const (&at)[8]) {
  asm volatile(
      "ds_read_b64_tr_b8 %0, %8\n\tds_read_b64_tr_b8 %1, %9\n\t"
      "ds_read_b64_tr_b8 %2, %10\n\tds_read_b64_tr_b8 %3, %11\n\t"
      "ds_read_b64_tr_b8 %4, %12\n\tds_read_b64_tr_b8 %5, %13\n\t"
      "ds_read_b64_tr_b8 %6, %14\n\tds_read_b64_tr_b8 %7, %15\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]),
        "=&v"(v[6]), "=&v"(v[7])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "v"(at[4]), "v"(at[5]), "v"(at[6]),
        "v"(at[7])
      : "memory");
}
__device__ __forceinline__ void read_transposed4x8(u32x2 (&v)[4], const LDS char *const (&at)[4]) {
  asm volatile(
      "ds_read_b64_tr_b8 %0, %4\n\tds_read_b64_tr_b8 %1, %5\n\t"
      "ds_read_b64_tr_b8 %2, %6\n\tds_read_b64_tr_b8 %3, %7\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
      : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
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

// Of 8-bit values NaN (0x7F and 0xFF), and under the largest scale, of which no larger is looked up
// (scale_exponent), those from 256 on (0x78): bit 7 of each byte that is one.
template <typename T>
__device__ __forceinline__ uint32_t odd_bytes(uint32_t v, float scale) {
  const bool largest = __float_as_uint(scale) >> 23 == 127 + kScaleMost<T>;
  return ((v & 0x7F7F7F7Fu) + (largest ? 0x08080808u : 0x01010101u)) & 0x80808080u;
}
// v without them; `any`: there were some, in the wave.
template <typename T>
__device__ __forceinline__ u32x2 finite_bytes(u32x2 v, float lo, float hi, bool &any) {
  const u32x2 s = {odd_bytes<T>(v[0], lo), odd_bytes<T>(v[1], hi)};
  if (__builtin_expect(__any((s[0] | s[1]) != 0), 0)) {
    any = true;
#pragma unroll
    for (int i = 0; i < 2; ++i) v[i] &= ~(s[i] | (s[i] - (s[i] >> 7)));
  }
  return v;
}

// Eight values of 8 bits (the type's own conversions, exact: four significant bits times a power of
// two that keeps them normal, or whole steps of fp16's smallest).  The scale's exponent counts.
__device__ __forceinline__ u32x4 from_e4m3(BF16, u32x2 w, float lo, float hi) {
  return u32x4{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], lo, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], lo, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], hi, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], hi, true))};
}
__device__ __forceinline__ u32x4 from_e4m3(FP16, u32x2 w, float lo, float hi) {
  return u32x4{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], lo, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[0], lo, true)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], hi, false)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[1], hi, true))};
}

// Place among the scales of keys of the block of 16 positions that holds position p of page
// `page`, at key-value head kv; those of values come page_size / kScaleKeys later.
__device__ __forceinline__ int64_t scale_place(const Attention &a, int page, int kv, int p) {
  const int blocks = 1 << (a.batch.page_shift - kScaleShift);
  return page * a.scale_stride + 2 * kv * blocks + ((p >> kScaleShift) & (blocks - 1));
}

// Exponents of a block's two scales: of keys in the low byte, of values in the next.  None is
// beyond those of the append, whatever lies in the scales of pages that nobody uses.
template <typename T>
__device__ __forceinline__ uint32_t scale_exponent(float s) {
  return min(__float_as_uint(s) >> 23 & 0xFFu, (uint32_t)(127 + kScaleMost<T>));
}
template <typename T>
__device__ __forceinline__ uint32_t load_exponents(const Attention &a, int page, int kv, int p) {
  const float *scale = a.scales + scale_place(a, page, kv, p);
  const float k = scale[0], v = scale[1 << (a.batch.page_shift - kScaleShift)];
  return scale_exponent<T>(k) | scale_exponent<T>(v) << 8;
}
__device__ __forceinline__ float key_scale(uint32_t e) { return __uint_as_float((e & 0xFFu) << 23); }
__device__ __forceinline__ float value_scale(uint32_t e) {
  return __uint_as_float((e & 0xFF00u) << 15);
}

// The value row of a key at the key-value head whose rows begin at `head`, for the infinities and
// NaN among its channels.
template <typename T, int D, typename C>
struct ValueRow {
  const typename Cache<C>::Elem *row;
  float scale;
  __device__ __forceinline__ ValueRow(const Attention &a, int s, int kv, int64_t head, int k) {
    const int page = paged_number(a.batch, s, k);
    row = static_cast<const typename Cache<C>::Elem *>(a.v_pages) + page * a.batch.page_stride +
          head + (int64_t)(k & ((1 << a.batch.page_shift) - 1)) * D;
    if constexpr (Cache<C>::kScaled)
      scale = value_scale(load_exponents<T>(a, page, kv, k));
  }
  // those among the four channels from d, 0 for others
  __device__ __forceinline__ f32x4 odd_parts(int d) const {
    u32x2 w;
    if constexpr (Cache<C>::kScaled) {
      const uint32_t v = ldg<uint32_t>(row + d);
      const u32x4 x = from_e4m3(T{}, u32x2{v, v}, scale, scale);
      w = u32x2{x[0], x[1]};
    } else {
      const uint2 v = ldg_u2(row + d);
      w = u32x2{v.x, v.y};
    }
    return f32x4{Pair<T>::odd_part(w[0] & 0xFFFFu), Pair<T>::odd_part(w[0] >> 16),
                 Pair<T>::odd_part(w[1] & 0xFFFFu), Pair<T>::odd_part(w[1] >> 16)};
  }
};

// ------------------------------------------------------------------ shares of keys
// The keys of the sequences with few rows, in blocks of 64 and one sequence after another,
// are cut into `shares` equal spans, one for each workgroup of a key-value head: as much
// work for each, whatever the lengths.  Every workgroup works the cuts out from the lengths,
// so the host needs to know none of them and a captured call follows them.  Blocks of 8-bit keys
// are twice as long, as a wave's steps are.
template <typename C, int W>
constexpr int kBlockKeys = W * Cache<C>::kFewKeys;

// count > 0 of a sequence whose rows fit the few-row kernel
__device__ __forceinline__ bool few_rows(const PagedSequence &q, int group) {
  return q.count > 0 && q.count <= kFewRows / group;
}
// Blocks of a sequence: 0 of one that is not the few-row kernel's, at least 1 of others.
template <typename C, int W>
__device__ __forceinline__ int few_blocks(const Attention &a, const PagedSequence &q) {
  return few_rows(q, a.group) ? max((q.length + kBlockKeys<C, W> - 1) / kBlockKeys<C, W>, 1) : 0;
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

// The lane's sequence, of up to 64; of more, none.
__device__ __forceinline__ PagedSequence lane_sequence(const Attention &a) {
  const int S = a.batch.sequences;
  return S <= 64 ? paged_sequences(a.batch, min((int)threadIdx.x & 63, S - 1), a.tokens)
                 : PagedSequence{};
}

// The spans, and the sequence that holds the first block of span `index`.  All threads of
// the W waves; scratch (2 W words of LDS) and found are free again afterwards.
template <typename C, int W>
__device__ Spans find_span(const Attention &a, int index, const PagedSequence &mine,
                           int64_t *scratch, Find *found, Find &got) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = a.batch.sequences;
  Spans sp;
  got = {0, -1};
  auto blocks = [&](int s) {
    return s < S ? few_blocks<C, W>(a, paged_sequences(a.batch, s, a.tokens)) : 0;
  };
  if (S <= 64) {  // every wave by itself: a sequence a lane
    const uint32_t n = lane < S ? few_blocks<C, W>(a, mine) : 0;  // 64 of at most 2^25
    const uint32_t sum = wave_scan(n);
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
  const int own = blocks(tid);
  int64_t all = own;
  for (int s = tid + W * 64; s < S; s += W * 64) all += blocks(s);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) all += __shfl_xor(all, o, 64);
  if (lane == 0) scratch[wave] = all;
  __syncthreads();
  sp.blocks = 0;
  for (int w = 0; w < W; ++w) sp.blocks += scratch[w];
  sp.spans = (int)min((int64_t)a.shares, sp.blocks);
  if (index < sp.spans) {
    const int64_t want = sp.start(index);
    int64_t base = 0;  // blocks before this group of sequences
    for (int c = 0; c < S && base <= want; c += W * 64) {
      const int n = c == 0 ? own : blocks(c + tid);
      const int64_t sum = (int64_t)wave_scan((uint64_t)n);
      __syncthreads();
      if (lane == 63) scratch[W + wave] = sum;
      __syncthreads();
      int64_t before = base + sum - n;
      for (int w = 0; w < W; ++w) {
        if (w < wave) before += scratch[W + w];
        base += scratch[W + w];
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
constexpr int kFewWaves = 4;  // W, but for attention_both_kernel with heads of 256

// Steps of 16 keys in a wave's ring: 64 KB for a workgroup, two of which share a CU, or 32 KB
// with heads of 64, of which three do: of 24 sequences of 300 to 5000 keys 33 instead of 37 us,
// of 200 up to 1000 keys 69 instead of 77 (16 heads each), one of 100000 keys 25 instead of
// 23.5.  Four workgroups, or three with 48 KB, took 1 to 5 % more than three with 32.
template <int D>
constexpr int few_steps() { return D == 256 ? 1 : 2; }
template <int D, int STEPS = few_steps<D>()>
constexpr int few_ring() { return STEPS * 2 * 16 * D * 2; }
template <int D, int W>
constexpr int few_merge() { return W * (kFewRows * (D + 4) + 2 * kFewRows) * 4; }
template <int D, int STEPS = few_steps<D>(), int W = kFewWaves>
constexpr int few_lds() {
  return W * few_ring<D, STEPS>() > few_merge<D, W>() ? W * few_ring<D, STEPS>() : few_merge<D, W>();
}

// The running state of a wave's 16 columns (column lane & 15 in each 16 lanes).
template <int D>
struct FewState {
  float m = -INFINITY, l = 0.0f;  // l: this lane's keys only
  f32x4 o[D / 16] = {};           // channels 16 i + 4 (lane >> 4) .. + 3
  bool odd = false;               // infinities or NaN were left out
};

// Scores of 16 keys, from row `row` of a tile in LDS, with the columns: keys 4 g .. 4 g + 3 a lane.
// A lane's 16 bytes of 8-bit keys are operands of two products, whose channels the queries follow
// (few_channel).
template <typename T, int D, typename C>
__device__ __forceinline__ f32x4 few_products(const LDS char *kt, int row, int base, float k_scale,
                                              const u32x4 (&q)[D / 32]) {
  constexpr int B = D * Cache<C>::kBytes;
  f32x4 s[2] = {};
  if constexpr (Cache<C>::kScaled) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const u32x4 k = *(const LDS u32x4 *)(kt + swizzled<B, kRows>(base, row, i * 4));
      s[0] = mfma16(T{}, from_e4m3(T{}, u32x2{k[0], k[1]}, k_scale, k_scale), q[2 * i], s[0]);
      s[1] = mfma16(T{}, from_e4m3(T{}, u32x2{k[2], k[3]}, k_scale, k_scale), q[2 * i + 1], s[1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const u32x4 k = *(const LDS u32x4 *)(kt + swizzled<B, kRows>(base, row, i * 4));
      s[i & 1] = mfma16(T{}, k, q[i], s[i & 1]);
    }
  }
  return s[0] + s[1];
}

// First of the eight channels of operand i of a lane's query.
template <typename C>
__device__ __forceinline__ int few_channel(int i, int g) {
  return Cache<C>::kScaled ? i / 2 * 64 + g * 16 + i % 2 * 8 : i * 32 + g * 8;
}

// Weights of a step's keys, packed: 4 g .. 4 g + 3 of each 16.
template <int KEYS>
struct FewWeights {
  uint32_t w[KEYS / 8];
};

// Exponents of the scales of a step's keys, of each 16.
template <typename C>
struct FewScales {
  uint32_t exponents[Cache<C>::kFewKeys / 16];
};

// Products of one step with the columns.
template <typename T, int D, typename C>
__device__ __forceinline__ FewWeights<Cache<C>::kFewKeys> few_scores(
    const LDS char *kt, const u32x4 (&q)[D / 32], int key0, int limit, float scale2,
    const FewScales<C> &scales, FewState<D> &st, int lane) {
  constexpr int B = D * Cache<C>::kBytes, N = Cache<C>::kFewKeys / 16;
  const int g = lane >> 4, r = lane & 15;
  const int base = opaque(r * B + ((g ^ swizzle<B>(r)) << 4));
  float x[N][4], mx = -INFINITY;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const f32x4 s = few_products<T, D, C>(kt, n * 16, base, key_scale(scales.exponents[n]), q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[n][i] = key0 + n * 16 + g * 4 + i < limit ? s[i] : -INFINITY;
      mx = fmaxf(mx, x[n][i]);
    }
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
  FewWeights<Cache<C>::kFewKeys> p;
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[n][i] = exp2_hw(__builtin_fmaf(x[n][i], scale2, -at));
      st.l += x[n][i];
    }
    p.w[2 * n] = T::pack2(x[n][0], x[n][1]);
    p.w[2 * n + 1] = T::pack2(x[n][2], x[n][3]);
  }
  return p;
}

// The values of a step as they lie in the cache: four keys of each 16th channel.
template <int D>
__device__ __forceinline__ void few_operands(const LDS char *vt, u32x2 (&v)[D / 16], int lane) {
  const int base = opaque(transpose_base<D * 2, kRows>((lane >> 4) * 4, 0, lane));
  constexpr int N = D == 64 ? 4 : 8;
  const LDS char *at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) at[i] = vt + swizzled<D * 2, kRows>(base, 0, i * 2);
  if constexpr (D == 64) {
    read_transposed4(v, at);
  } else {
    read_transposed8<0>(*reinterpret_cast<u32x2(*)[8]>(&v[0]), at);
    if constexpr (D == 256) read_transposed8<256>(*reinterpret_cast<u32x2(*)[8]>(&v[8]), at);
  }
}
// Of 8 bits, eight keys of each 16th channel, eight of them from 16 `first` on (four of heads of 64).
template <int D, int N>
__device__ __forceinline__ void few_operands8(const LDS char *vt, int first, u32x2 (&v)[N], int lane) {
  const int base = opaque(transpose8_base<D, kHalves, 16>((lane >> 4) * 4, 0, lane));
  const LDS char *at[N];
#pragma unroll
  for (int i = 0; i < N; ++i) at[i] = vt + swizzled<D, kHalves>(base, 0, first + i);
  if constexpr (N == 4)
    read_transposed4x8(v, at);
  else
    read_transposed8x8(v, at);
}

// Adds the weighted values of a step; `mixed`: some row does not see all its keys.
template <typename T, int D, typename C>
__device__ __forceinline__ void few_values(const LDS char *vt,
                                           const FewWeights<Cache<C>::kFewKeys> &p,
                                           const FewScales<C> &scales, bool mixed,
                                           FewState<D> &st, int lane) {
  if constexpr (Cache<C>::kScaled) {
    constexpr int N = D == 64 ? 4 : 8;
    const u32x4 w = {p.w[0], p.w[1], p.w[2], p.w[3]};
    const float lo = value_scale(scales.exponents[0]), hi = value_scale(scales.exponents[1]);
#pragma unroll
    for (int i0 = 0; i0 < D / 16; i0 += N) {
      u32x2 v[N];
      few_operands8<D, N>(vt, i0, v, lane);
      if (mixed) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const u32x2 x = finite_bytes<T>(v[i], lo, hi, st.odd);
          st.o[i0 + i] = mfma16(T{}, from_e4m3(T{}, x, lo, hi), w, st.o[i0 + i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          st.o[i0 + i] = mfma16(T{}, from_e4m3(T{}, v[i], lo, hi), w, st.o[i0 + i]);
      }
    }
  } else {
    uint32_t any = 0;
    u32x2 v[D / 16];
    few_operands<D>(vt, v, lane);
    const u32x2 w = {p.w[0], p.w[1]};
    if (mixed) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        v[i] = u32x2{Pair<T>::finite(v[i][0], any), Pair<T>::finite(v[i][1], any)};
      st.odd |= __any(any != 0);
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) st.o[i] = mfma16k16(T{}, v[i], w, st.o[i]);
  }
}

// The keys of a wave: steps of kFewKeys keys, `stride` steps apart, and the pages they lie in.
template <typename C>
struct FewKeys {
  const typename Cache<C>::Elem *k, *v;  // of the key-value head, in page 0
  const int32_t *table;
  int64_t page_stride;
  int shift, pages, entries;
  int first, stride, steps;  // first step's number, and how many
  int page_of;               // pages of 64 times 16 keys (kSteps steps), one a lane
  uint32_t exponents;        // of 8 bits: their scales'
  static constexpr int kUnits = Cache<C>::kFewKeys / 16, kSteps = 64 / kUnits;
};

// The lane's key among those of the steps from `from` on, its entry of the page table, and what
// that gives: the page, and of 8 bits the scales.
template <typename C>
__device__ __forceinline__ int few_key(const FewKeys<C> &f, int from, int lane) {
  constexpr int U = FewKeys<C>::kUnits;
  const int step = f.first + min(from + lane / U, max(f.steps - 1, 0)) * f.stride;
  return step * Cache<C>::kFewKeys + lane % U * 16;
}
template <typename C>
__device__ __forceinline__ int few_entry(const FewKeys<C> &f, int from, int lane) {
  return f.table[min(few_key(f, from, lane) >> f.shift, f.entries - 1)];
}
template <typename T, typename C>
__device__ __forceinline__ void few_pages(const Attention &a, FewKeys<C> &f, int entry, int from,
                                          int kv, int lane) {
  f.page_of = clamp_index32(entry, f.pages);
  settle(f.page_of);
  if constexpr (Cache<C>::kScaled)
    f.exponents = load_exponents<T>(a, f.page_of, kv, few_key(f, from, lane));
}

// Loads step i's rows of one side (a step past the end: again the last, never used).
template <int D, typename C, Swizzle S>
__device__ __forceinline__ void few_load(const FewKeys<C> &f, const typename Cache<C>::Elem *side,
                                         int i, LDS char *to, int lane) {
  constexpr int U = FewKeys<C>::kUnits, B = D * Cache<C>::kBytes;
  const int j = min(i, f.steps - 1), key0 = (f.first + j * f.stride) * Cache<C>::kFewKeys;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int key = key0 + u * 16;
    const int page = __builtin_amdgcn_readlane(f.page_of, (j * U + u) & 63);
    const auto *src = side + page * f.page_stride + (int64_t)(key & ((1 << f.shift) - 1)) * D;
    load_rows<B, 16, S, kStream>(src, u * 16, to + u * 16 * B, lane);
  }
}

// The transpose reads of 8-bit values touch other rows together than those of 16 bits.
template <typename C>
constexpr Swizzle kFewValues = Cache<C>::kScaled ? kHalves : kRows;

// Step i, from its place in the ring, which is refilled as soon as it is read; the counts of
// loads that may still be out are stated here.  `scales`: the step's, looked up before the pages
// of the steps that it loads.
template <typename C>
__device__ __forceinline__ FewScales<C> few_step_scales(const FewKeys<C> &f, int i) {
  FewScales<C> s = {};
  if constexpr (Cache<C>::kScaled)
#pragma unroll
    for (int u = 0; u < FewKeys<C>::kUnits; ++u)
      s.exponents[u] = __builtin_amdgcn_readlane(f.exponents, (i * FewKeys<C>::kUnits + u) & 63);
  return s;
}
template <typename T, int D, typename C, int STEPS>
__device__ __forceinline__ void few_step(LDS char *ring, const FewKeys<C> &f,
                                         const FewScales<C> &scales, const u32x4 (&q)[D / 32],
                                         int i, int limit, int all_see, float scale2,
                                         FewState<D> &st, int lane) {
  constexpr int KEYS = Cache<C>::kFewKeys;
  constexpr int TILE = KEYS * D * Cache<C>::kBytes, N = TILE / 1024;  // bytes, loads of one side
  constexpr int OUT = (2 * STEPS - 1) * N;
  LDS char *k = ring + i % STEPS * 2 * TILE, *v = k + TILE;
  const int key = (f.first + i * f.stride) * KEYS;
  wait_loads<OUT>();
  const auto p = few_scores<T, D, C>(k, q, key, limit, scale2, scales, st, lane);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  few_load<D, C, kRows>(f, f.k, i + STEPS, k, lane);
  wait_loads<OUT>();
  few_values<T, D, C>(v, p, scales, key + KEYS > all_see, st, lane);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  few_load<D, C, kFewValues<C>>(f, f.v, i + STEPS, v, lane);
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
template <typename T, int D, typename C, int STEPS, int W>
__device__ __forceinline__ void few_part(const Attention &a, const PagedSequence &seq, int s, int kv,
                                         int b0, int b1, int64_t part, char *lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = seq.count * a.group;
  const int col = min(lane & 15, rows - 1), g = lane >> 4;
  const RowPlace at = row_place(a, seq, kv, col);
  u32x4 q[D / 32];

  using Elem = typename Cache<C>::Elem;
  constexpr int KEYS = Cache<C>::kFewKeys;
  FewKeys<C> f;
  const int64_t head = (int64_t)(kv << a.batch.page_shift) * D;
  f.k = static_cast<const Elem *>(a.k_pages) + head;
  f.v = static_cast<const Elem *>(a.v_pages) + head;
  f.table = a.batch.table + s * a.batch.table_stride;
  f.page_stride = a.batch.page_stride, f.shift = a.batch.page_shift;
  f.pages = a.batch.pages, f.entries = a.batch.table_pages;
  const int last = min(b1 * (kBlockKeys<C, W> / KEYS), (seq.length + KEYS - 1) / KEYS);
  f.first = b0 * (kBlockKeys<C, W> / KEYS) + wave, f.stride = W;
  f.steps = last > f.first ? (last - f.first + W - 1) / W : 0;
  const int limit = min(seq.base + col / a.group + 1, seq.length);
  const int all_see = min(seq.base + 1, seq.length);  // keys that every row sees

  FewState<D> st;
  if (f.steps > 0) {
    // The pages' and the queries' loads go out together, the rows' behind the pages', and only then
    // are the others waited for.
    int entry = few_entry(f, 0, lane);
    const uint16_t *qr = a.q + (int64_t)at.token * a.q_token + (int64_t)at.head * a.q_head;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) q[i] = ldg16(qr + few_channel<C>(i, g));
    __builtin_amdgcn_sched_barrier(0);
    settle(entry);
    few_pages<T>(a, f, entry, 0, kv, lane);
    LDS char *ring = (LDS char *)lds + wave * few_ring<D, STEPS>();
    constexpr int TILE = KEYS * D * Cache<C>::kBytes;
    static_assert(TILE * 2 * STEPS == few_ring<D, STEPS>(), "a ring holds its steps");
    FewScales<C> scales[STEPS];
    for (int j = 0; j < STEPS; ++j) {  // in this order: the waits count what was issued later
      few_load<D, C, kRows>(f, f.k, j, ring + 2 * j * TILE, lane);
      asm volatile("" ::: "memory");
      few_load<D, C, kFewValues<C>>(f, f.v, j, ring + (2 * j + 1) * TILE, lane);
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      settle(q[i]);
      q[i] ^= a.flip;
    }
    if constexpr (Cache<C>::kScaled) settle(f.exponents);
#pragma unroll
    for (int j = 0; j < STEPS; ++j) scales[j] = few_step_scales(f, j);
    for (int i = 0; i < f.steps; ++i) {
      if (((i + STEPS) & (FewKeys<C>::kSteps - 1)) == 0) {  // that step is loaded next
        few_pages<T>(a, f, few_entry(f, i + STEPS, lane), i + STEPS, kv, lane);
        if constexpr (Cache<C>::kScaled) settle(f.exponents);
      }
      const FewScales<C> now = scales[0];
#pragma unroll
      for (int j = 1; j < STEPS; ++j) scales[j - 1] = scales[j];
      scales[STEPS - 1] = few_step_scales(f, i + STEPS);
      few_step<T, D, C, STEPS>(ring, f, now, q, i, limit, all_see, a.scale2, st, lane);
    }
    wait_loads<0>();  // the last refills, before the ring is used otherwise
    if (__builtin_expect(st.odd, 0)) {
      for (int i = 0; i < f.steps; ++i) {
        const int key = (f.first + i * f.stride) * KEYS;
        if (key + KEYS <= all_see) continue;
        for (int k = key; k < min(key + KEYS, limit); ++k) {
          const ValueRow<T, D, C> v(a, s, kv, head, k);
#pragma unroll
          for (int j = 0; j < D / 16; ++j) st.o[j] += v.odd_parts(j * 16 + g * 4);
        }
      }
    }
  }

  // The waves' sums, scaled to the largest of their maxima.
  __syncthreads();
  float *sums = reinterpret_cast<float *>(lds);  // [wave][row][D + 4]
  float *ml = sums + W * kFewRows * (D + 4);  // [wave][row] maxima, then sums
  st.l = across32(across16(st.l, Add()), Add());
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    *reinterpret_cast<f32x4 *>(sums + (wave * kFewRows + (lane & 15)) * (D + 4) + i * 16 + g * 4) =
        st.o[i];
  if (lane < 16) {
    ml[wave * kFewRows + lane] = st.m;
    ml[(W + wave) * kFewRows + lane] = st.l;
  }
  __syncthreads();
  for (int i = tid; i < rows * (D / 4); i += W * 64) {
    const int c = i / (D / 4), d = i % (D / 4) * 4;
    float m = ml[c], l = 0.0f;
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, ml[w * kFewRows + c]);
    f32x4 o = {};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float k = decay(ml[w * kFewRows + c], m);
      l += ml[(W + w) * kFewRows + c] * k;
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

// Workgroup `index` of those of few rows.
template <typename T, int D, typename C, int STEPS, int W>
__device__ __forceinline__ void few_span(const Attention &a, int index, const PagedSequence &mine,
                                         char *lds) {
  int64_t *scratch = reinterpret_cast<int64_t *>(lds);
  const int kv = index % a.batch.kv_heads, span = index / a.batch.kv_heads;
  Find at;
  const Spans sp = find_span<C, W>(a, span, mine, scratch, reinterpret_cast<Find *>(scratch + 2 * W), at);
  if (at.s < 0) return;
  int64_t block = sp.start(span);
  const int64_t end = sp.start(span + 1);
  int s = __builtin_amdgcn_readfirstlane(at.s);
  int done = __builtin_amdgcn_readfirstlane((int)(block - at.first));  // blocks of s before
  bool later = false;
  for (; block < end && s < a.batch.sequences; ++s, done = 0) {
    const PagedSequence seq = sequence_at(a.batch, s, mine, a.tokens);
    const int all = few_blocks<C, W>(a, seq);
    const int take = __builtin_amdgcn_readfirstlane((int)min((int64_t)(all - done), end - block));
    if (take <= 0) continue;
    if (done == 0 && threadIdx.x == 0)  // where its parts are, for the kernel that joins them
      a.parts[s * a.batch.kv_heads + kv] = {span, later, sp.of(block + all - 1) - span + 1};
    few_part<T, D, C, STEPS, W>(a, seq, s, kv, done, done + take,
                      take == all ? -1 : part_row(a, span, later, kv), lds);
    block += take;
    later = true;
  }
}

template <typename T, int D, typename C>
__global__ __launch_bounds__(256, Cache<C>::kScaled ? 2 : 1) void attention_few_kernel(Attention a) {
  // One array: with several, the compiler waits for all direct loads at each LDS read.
  __shared__ __attribute__((aligned(16))) char lds[few_lds<D>()];
  few_span<T, D, C, few_steps<D>(), kFewWaves>(a, blockIdx.x, lane_sequence(a), lds);
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
template <int D, typename C>
struct TileForm {
  static constexpr int kGroups = D == 256 ? 2 : 1, kSteps = D == 256 ? 1 : Cache<C>::kTileSteps;
  static constexpr int kWaves = 4 * kGroups, kKeys = 32 * kGroups * kSteps;
  static constexpr int kBytes = kKeys * D * Cache<C>::kBytes;  // of one side
};

// Tiles of the rows of a sequence, unless the few-row kernel takes them.
__device__ __forceinline__ int tile_count(const Attention &a, const PagedSequence &q) {
  if (a.few && few_rows(q, a.group)) return 0;
  return (int)(((int64_t)q.count * a.group + kTileRows - 1) / kTileRows);
}

// Keys that the last row of a sequence's tile sees, the most of its rows.
__device__ __forceinline__ int tile_keys(const PagedSequence &q, int group, int tile) {
  const int last = min((int64_t)(tile + 1) * kTileRows, (int64_t)q.count * group) - 1;
  return max(min(q.base + last / group + 1, q.length), 0);
}

// Keys of n tiles of a sequence together (their mean is that of the first and the last).
__device__ __forceinline__ uint64_t all_keys(const Attention &a, const PagedSequence &q, int n) {
  if (n == 0) return 0;
  return ((uint64_t)tile_keys(q, a.group, 0) + tile_keys(q, a.group, n - 1)) * n / 2;
}

struct TilePlace {
  int s, tile;        // s < 0: none
  int split, splits;  // which part of its keys, of how many
};

// All tiles of a call, and their keys.
struct TileTotals {
  int tiles;
  uint64_t keys;
};

// Parts of a tile that sees `keys` keys, where sequences differ: about equal parts, as many as
// the tiles, which take one or more each, leave of so many rounds of workgroups that they fill
// two thirds at most; none below 256 keys.  Against as many parts for every tile, 12 sequences of
// up to 700 new tokens took 52 us instead of 61 (heads of 128) and 61 instead of 77 (256), 24 of
// 8 to 24 tokens 46 instead of 55; parts of 128 or 512 keys and fewer or more rounds took up to
// 30 % more in one case or another.
__device__ __forceinline__ int tile_parts(const Attention &a, const TileTotals &total, int keys) {
  const int rounds = (int)((float)total.tiles * 1.5f / (float)a.room) + 1;
  const float all = (float)max(total.keys, (uint64_t)1);
  const float n = (float)keys * (float)(rounds * a.room - total.tiles) / all + 0.5f;
  return max(min(min((int)fminf(n, 65536.0f), a.splits), keys / 256), 1);
}
// A sequence's tiles have as many places each in the grid as its last one, which sees the most keys,
// has parts, so that few places are empty.  Workgroups go to the chip's dies and CUs in turn, and
// with `splits` places for every tile those of the parts that there are came round to the same
// CUs: 2048 new tokens beside 8 of one (heads of 128) took 141 us instead of 95, behind 8192 keys
// beside 32 (256) 1022 instead of 377.  A grid of all first parts, then all second ones, has the
// empty places before work: 12 sequences of up to 700 new tokens 50 us instead of 45.
__device__ __forceinline__ int tile_places(const Attention &a, const TileTotals &total,
                                           const PagedSequence &q, int n) {
  return n > 0 ? tile_parts(a, total, tile_keys(q, a.group, n - 1)) : 1;
}
// Place `at` of a sequence's n tiles with `places` each; a tile's first part is at another one in
// each, for the same reason.
__device__ __forceinline__ TilePlace tile_place(const Attention &a, const TileTotals &total, int s,
                                                const PagedSequence &q, int n, int places, int at) {
  const int t = at / places, tile = n - 1 - t;
  return {s, tile, (at % places + t + (t >> 2) + (t >> 4)) % places,
          tile_parts(a, total, tile_keys(q, a.group, tile))};
}

// The index-th tile, or place of one, and its sequence; the tile with the most keys of a sequence
// comes first.  `split`: the part, where all tiles have a.splits.  All THREADS threads; scratch (a
// word and a long word a wave) and found are free again afterwards.
template <int THREADS>
__device__ TilePlace find_tile(const Attention &a, int index, int split, const PagedSequence &mine,
                               int *scratch, uint64_t *sums, TilePlace *found,
                               PagedSequence &seq) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = a.batch.sequences;
  const bool places = a.room > 0;
  if (S <= 64) {  // each wave for itself
    const int n = lane < S ? tile_count(a, mine) : 0;
    TileTotals total = {};
    int m = 1;
    if (places) {
      total = {(int)wave_total((uint64_t)n), wave_total(all_keys(a, mine, n))};
      m = tile_places(a, total, mine, n);
    }
    const int sum = (int)wave_scan((uint32_t)(n * m));
    const uint64_t hit = __ballot(index >= sum - n * m && index < sum);
    if (!hit) return {-1, 0, 0, 0};
    const int at = __builtin_ctzll(hit), before = __builtin_amdgcn_readlane(sum - n * m, at);
    const int tiles = __builtin_amdgcn_readlane(n, at);
    seq = sequence_at(a.batch, at, mine, a.tokens);
    if (!places) return {at, tiles - 1 - (index - before), split, a.splits};
    return tile_place(a, total, at, seq, tiles, __builtin_amdgcn_readlane(m, at), index - before);
  }
  if (tid == 0) found->s = -1;
  TileTotals total = {};
  if (places) {
    for (int c = tid; c < S; c += THREADS) {
      const PagedSequence q = paged_sequences(a.batch, c, a.tokens);
      const int n = tile_count(a, q);
      total.tiles += n, total.keys += all_keys(a, q, n);
    }
    total.tiles = (int)wave_total((uint64_t)total.tiles), total.keys = wave_total(total.keys);
    if (lane == 0) scratch[wave] = total.tiles, sums[wave] = total.keys;
    __syncthreads();
    total = {};
    for (int w = 0; w < THREADS / 64; ++w) total.tiles += scratch[w], total.keys += sums[w];
  }
  int base = 0;
  for (int c = 0; c < S && base <= index; c += THREADS) {
    const PagedSequence q = paged_sequences(a.batch, min(c + tid, S - 1), a.tokens);
    const int n = c + tid < S ? tile_count(a, q) : 0;
    const int m = places ? tile_places(a, total, q, n) : 1;
    const int sum = (int)wave_scan((uint32_t)(n * m));
    __syncthreads();
    if (lane == 63) scratch[wave] = sum;
    __syncthreads();
    int before = base;
    for (int w = 0; w < THREADS / 64; ++w) {
      if (w < wave) before += scratch[w];
      base += scratch[w];
    }
    before += sum - n * m;
    if (index >= before && index < before + n * m)
      *found = places ? tile_place(a, total, c + tid, q, n, m, index - before)
                      : TilePlace{c + tid, n - 1 - (index - before), split, a.splits};
  }
  __syncthreads();
  const TilePlace got = *found;
  __syncthreads();
  if (got.s >= 0) seq = sequence_at(a.batch, got.s, {}, a.tokens);
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
template <typename C>
struct TilePages {
  const int32_t *table;
  int64_t page_stride;
  const typename Cache<C>::Elem *k, *v;  // of the key-value head, in page 0
  int shift, pages, entries;
  int from, page_of;
  int scaled;          // first key of the exponents
  uint32_t exponents;  // of 8 bits: their scales'; in the upper half those of the pages from `from`
                       // on, until the tile there is next (its rows are loaded a tile earlier)
};

// The lane's entry of the page table for the keys from `key` on, and what that gives: the page, and
// of 8 bits the scales.
template <typename C>
__device__ __forceinline__ int tile_entry(const TilePages<C> &f, int key, int lane) {
  return f.table[min((key + lane * 16) >> f.shift, f.entries - 1)];
}
template <typename T, typename C>
__device__ __forceinline__ void tile_pages(const Attention &a, TilePages<C> &f, int entry, int key,
                                           int kv, int lane) {
  f.from = key;
  f.page_of = clamp_index32(entry, f.pages);
  settle(f.page_of);
  if constexpr (Cache<C>::kScaled)
    f.exponents = (f.exponents & 0xFFFFu) |
                  load_exponents<T>(a, f.page_of, kv, key + lane * 16) << 16;
}

// The transpose reads of 8-bit values touch other rows together than those of 16 bits.
template <typename C>
constexpr Swizzle kTileValues = Cache<C>::kScaled ? kOctets : kQuads;

// Loads a tile of keys and values from `key` on into LDS: ROWS rows of each a wave.
template <typename T, int D, int ROWS, typename C>
__device__ __forceinline__ void tile_load(const Attention &a, TilePages<C> &f, int key,
                                          LDS char *kt, LDS char *vt, int kv, int wave, int lane) {
  constexpr int B = D * Cache<C>::kBytes;
  if (key - f.from >= 1024) {
    tile_pages<T>(a, f, tile_entry(f, key, lane), key, kv, lane);
    if constexpr (Cache<C>::kScaled) settle(f.exponents);
  }
#pragma unroll
  for (int r = 0; r < ROWS; r += 16) {  // of one page each
    constexpr int N = ROWS < 16 ? ROWS : 16;
    const int row = wave * ROWS + r, k = key + row, to = row * B;
    const int page = __builtin_amdgcn_readlane(f.page_of, (k - f.from) >> 4);
    const int64_t at = page * f.page_stride + (int64_t)(k & ((1 << f.shift) - 1)) * D;
    load_rows<B, N>(f.k + at, row, kt + to, lane);
    load_rows<B, N, kTileValues<C>>(f.v + at, row, vt + to, lane);
  }
}

// The exponents that belong to the tile at `key`, before the next one's pages are looked up.
template <typename C>
__device__ __forceinline__ void tile_advance(TilePages<C> &f, int key) {
  if constexpr (Cache<C>::kScaled)
    if (key == f.from) f.exponents >>= 16, f.scaled = key;
}

// Exponents of the scales of a step of 32 keys, `at` keys behind f.scaled: of keys 0 .. 15 and
// 16 .. 31.
struct TileScales {
  uint32_t exponents[2];
};
template <typename C>
__device__ __forceinline__ TileScales tile_scales(const TilePages<C> &f, int at) {
  TileScales s = {};
  if constexpr (Cache<C>::kScaled)
#pragma unroll
    for (int u = 0; u < 2; ++u)
      s.exponents[u] = __builtin_amdgcn_readlane(f.exponents, (at >> 4) + u);
  return s;
}

// Operands that are read from LDS before the product that needs the first of them.  Left to its
// own order, the compiler waits for each operand right before its product: 9 % more time with
// heads of 256 (2048 tokens behind 8192 keys: 374 us instead of 337), 3 % with 128.
constexpr int kAheadReads = 4;

// Operand of 16 keys from row `ks` of the tile, channels 32 i ..
template <typename T, int D, typename C>
__device__ __forceinline__ u32x4 tile_operand(const LDS char *vt, int base, int i, int ks) {
  const u32x2 lo = read_transposed<D * 2, kQuads>(vt, base, ks, i * 32);
  const u32x2 hi = read_transposed<D * 2, kQuads>(vt, base, ks + 8, i * 32);
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// Adds the weighted values of 32 keys; MIXED: some row does not see all of them.
template <typename T, int D, bool MIXED>
__device__ __forceinline__ void tile_values(T, const LDS char *vt, const u32x4 (&p)[2],
                                            const TileScales &, TileState<D> &st, int lane) {
  const int base =
      opaque(transpose_base<D * 2, kQuads>((lane >> 5) * 4, ((lane >> 4) & 1) * 16, lane));
  if constexpr (MIXED) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        u32x4 v = tile_operand<T, D, T>(vt, base, i, ks * 16);
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
  for (int u = 0; u < kAheadReads; ++u) v[u] = tile_operand<T, D, T>(vt, base, u / 2, u % 2 * 16);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int u = 0; u < D / 16; ++u) {
    st.o[u / 2] = mfma32(T{}, v[u % kAheadReads], p[u % 2], st.o[u / 2]);
    const int n = u + kAheadReads;
    if (n < D / 16) v[u % kAheadReads] = tile_operand<T, D, T>(vt, base, n / 2, n % 2 * 16);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
}

// The same of 8 bits: a read is an operand of two channels' 16 keys, converted a product ahead.
template <typename T, int D, bool MIXED>
__device__ __forceinline__ void tile_values(E4M3, const LDS char *vt, const u32x4 (&p)[2],
                                            const TileScales &scales, TileState<D> &st,
                                            int lane) {
  const float scale[2] = {value_scale(scales.exponents[0]), value_scale(scales.exponents[1])};
  const int base =
      opaque(transpose8_base<D, kOctets, 8>((lane >> 5) * 4, (lane >> 4) & 1, lane));
  auto read = [&](int u) {
    return read_transposed8b<D, kOctets>(vt, base, u % 2 * 16, u / 2 * 2);
  };
  if constexpr (MIXED) {
#pragma unroll
    for (int u = 0; u < D / 16; ++u) {
      const float own = scale[u % 2];
      const u32x2 v = finite_bytes<T>(read(u), own, own, st.odd);
      st.o[u / 2] = mfma32(T{}, from_e4m3(T{}, v, own, own), p[u % 2], st.o[u / 2]);
    }
    return;
  }
  __builtin_amdgcn_s_setprio(1);
  u32x2 raw[kAheadReads];
#pragma unroll
  for (int u = 0; u < kAheadReads; ++u) raw[u] = read(u);
  __builtin_amdgcn_sched_barrier(0);
  u32x4 v = from_e4m3(T{}, raw[0], scale[0], scale[0]);
#pragma unroll
  for (int u = 0; u < D / 16; ++u) {
    st.o[u / 2] = mfma32(T{}, v, p[u % 2], st.o[u / 2]);
    if (u + kAheadReads < D / 16) raw[u % kAheadReads] = read(u + kAheadReads);
    if (u + 1 < D / 16)
      v = from_e4m3(T{}, raw[(u + 1) % kAheadReads], scale[(u + 1) % 2], scale[(u + 1) % 2]);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
}

// Scores of 32 keys with a wave's 32 rows.
template <typename T, int D>
__device__ __forceinline__ f32x16 tile_products(T, const LDS char *kt, const u32x4 (&q)[D / 16],
                                                const TileScales &, int lane) {
  const int h = lane >> 5, r = lane & 31;
  const int base = opaque(r * (D * 2) + ((h ^ swizzle<D * 2>(r)) << 4));
  f32x16 x = {};
  auto read = [&](int i) {
    return *(const LDS u32x4 *)(kt + swizzled<D * 2, kRows>(base, 0, i * 2));
  };
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
  return x;
}

// The same of 8 bits: a read is the operands of two products (tile_channel), each converted a
// product ahead.
template <typename T, int D>
__device__ __forceinline__ f32x16 tile_products(E4M3, const LDS char *kt, const u32x4 (&q)[D / 16],
                                                const TileScales &scales, int lane) {
  constexpr int READS = D / 32, AHEAD = READS < 4 ? READS : 4;
  const int h = lane >> 5, r = lane & 31;
  const int base = opaque(r * D + ((h ^ swizzle<D>(r)) << 4));
  const float own = key_scale(r < 16 ? scales.exponents[0] : scales.exponents[1]);
  f32x16 x = {};
  auto read = [&](int i) {
    return *(const LDS u32x4 *)(kt + swizzled<D, kRows>(base, 0, i * 2));
  };
  u32x4 raw[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) raw[i] = read(i);
  __builtin_amdgcn_sched_barrier(0);
  auto operand = [&](int i) {
    const u32x4 k = raw[i / 2 % AHEAD];
    return from_e4m3(T{}, i % 2 ? u32x2{k[2], k[3]} : u32x2{k[0], k[1]}, own, own);
  };
  u32x4 k = operand(0);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    x = mfma32(T{}, k, q[i], x);
    if (i + 1 < D / 16) k = operand(i + 1);
    if (i % 2 == 0 && i / 2 + AHEAD < READS) raw[i / 2 % AHEAD] = read(i / 2 + AHEAD);
    __builtin_amdgcn_sched_barrier(0);
  }
  return x;
}

// First of the eight channels of operand i of a lane's query.
template <typename C>
__device__ __forceinline__ int tile_channel(int i, int h) {
  return Cache<C>::kScaled ? i / 2 * 32 + h * 16 + i % 2 * 8 : i * 16 + h * 8;
}

// 32 keys of a tile for a wave's 32 rows.  MIXED: some row does not see all of them.
// The wave's priority is raised while it feeds the matrix cores, so that the other wave of
// its SIMD does its softmax beside them.
template <typename T, int D, bool MIXED, typename C>
__device__ __forceinline__ void tile_step(const LDS char *kt, const LDS char *vt,
                                          const u32x4 (&q)[D / 16], int key, int limit,
                                          float scale2, const TileScales &scales,
                                          TileState<D> &st, int lane) {
  const int h = lane >> 5;
  __builtin_amdgcn_s_setprio(1);
  f32x16 x = tile_products<T, D>(C{}, kt, q, scales, lane);
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
  tile_values<T, D, MIXED>(C{}, vt, p, scales, st, lane);
}

// The waves' sums on their way out, half of the channels at a time: rows of D / 2 channels
// and a pad of four, then each row's maximum and sum.
template <int D>
constexpr int tile_pitch() { return D / 2 + 4; }
template <int D, typename C>
constexpr int tile_lds() {
  using F = TileForm<D, C>;
  constexpr int ring = 4 * F::kBytes, out = F::kWaves * 32 * (tile_pitch<D>() + 2) * 4;
  return out > ring ? out : ring;
}

// Workgroup (x, y) of those of tiles; y: the part, where all tiles have a.splits.
template <typename T, int D, typename C>
__device__ __forceinline__ void tile_rows(const Attention &a, int x, int y,
                                          const PagedSequence &mine, char *lds) {
  using F = TileForm<D, C>;
  using Elem = typename Cache<C>::Elem;
  constexpr int WAVES = F::kWaves, KEYS = F::kKeys, ROWS = KEYS / WAVES;
  constexpr int GROUPS = F::kGroups, TILE = F::kBytes, B = D * Cache<C>::kBytes;
  static_assert(GROUPS == 1 || GROUPS == 2, "two groups are joined");
  int *scratch = reinterpret_cast<int *>(lds);
  uint64_t *key_sums = reinterpret_cast<uint64_t *>(scratch + 8);
  TilePlace *found = reinterpret_cast<TilePlace *>(key_sums + 8);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int set = wave & 3, group = wave >> 2;
  const int kv = x % a.batch.kv_heads, index = x / a.batch.kv_heads;
  PagedSequence seq;
  const TilePlace place =
      find_tile<WAVES * 64>(a, index, y, mine, scratch, key_sums, found, seq);
  const int s = __builtin_amdgcn_readfirstlane(place.s);
  if (s < 0) return;
  const int tile = __builtin_amdgcn_readfirstlane(place.tile);
  const int rows = seq.count * a.group, c0 = tile * kTileRows;
  const int c = c0 + set * 32 + (lane & 31);
  const bool idle = c0 + set * 32 >= rows;
  const RowPlace at = row_place(a, seq, kv, min(c, rows - 1));
  const int limit = min(seq.base + min(c, rows - 1) / a.group + 1, seq.length);
  const int all_see = min(seq.base + c0 / a.group + 1, seq.length);  // seen by every row
  // keys that the tile's last row sees, and this part of them
  const int keys = tile_keys(seq, a.group, tile), tiles = (keys + KEYS - 1) / KEYS;
  const int split = __builtin_amdgcn_readfirstlane(place.split);
  const int splits = __builtin_amdgcn_readfirstlane(place.splits);
  if (split >= splits) return;
  const int key0 = (int)((int64_t)tiles * split / splits) * KEYS;
  const int key1 = min((int)((int64_t)tiles * (split + 1) / splits) * KEYS, keys);

  u32x4 q[D / 16];
  const uint16_t *qr = a.q + (int64_t)at.token * a.q_token + (int64_t)at.head * a.q_head;
  TileState<D> st;
  LDS char *base = (LDS char *)lds;
  const int64_t head = (int64_t)(kv << a.batch.page_shift) * D;
  if (key0 < key1) {
    TilePages<C> f;
    f.table = a.batch.table + s * a.batch.table_stride, f.page_stride = a.batch.page_stride;
    f.k = static_cast<const Elem *>(a.k_pages) + head;
    f.v = static_cast<const Elem *>(a.v_pages) + head, f.shift = a.batch.page_shift;
    f.pages = a.batch.pages, f.entries = a.batch.table_pages, f.exponents = 0;
    // The pages' and the queries' loads go out together, the rows' behind the pages', and only then
    // are the others waited for.
    int entry = tile_entry(f, key0, lane);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) q[i] = ldg16(qr + tile_channel<C>(i, lane >> 5));
    __builtin_amdgcn_sched_barrier(0);
    settle(entry);
    tile_pages<T>(a, f, entry, key0, kv, lane);
    tile_load<T, D, ROWS>(a, f, key0, base, base + TILE, kv, wave, lane);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      settle(q[i]);
      q[i] ^= a.flip;
    }
    if constexpr (Cache<C>::kScaled) settle(f.exponents);
    wait_loads<0>();
    __syncthreads();
    // A tile, the next one's loads started before it into the other half.
    int key = key0, half = 0;
    const int whole = min(key1, all_see);
    for (; key + KEYS <= whole; key += KEYS, half ^= 1) {
      LDS char *cur = base + half * 2 * TILE, *next = base + (half ^ 1) * 2 * TILE;
      tile_advance(f, key);
      if (key + KEYS < key1)
        tile_load<T, D, ROWS>(a, f, key + KEYS, next, next + TILE, kv, wave, lane);
      if (!idle)
#pragma unroll
        for (int i = 0; i < F::kSteps; ++i) {
          const int own = (i * GROUPS + group) * 32;
          tile_step<T, D, false, C>(cur + own * B, cur + TILE + own * B, q, key + own, limit,
                                    a.scale2, tile_scales(f, key + own - f.scaled), st, lane);
        }
      wait_loads<0>();
      __syncthreads();
    }
    for (; key < key1; key += KEYS, half ^= 1) {
      LDS char *cur = base + half * 2 * TILE, *next = base + (half ^ 1) * 2 * TILE;
      tile_advance(f, key);
      if (key + KEYS < key1)
        tile_load<T, D, ROWS>(a, f, key + KEYS, next, next + TILE, kv, wave, lane);
      if (!idle)
#pragma unroll
        for (int i = 0; i < F::kSteps; ++i) {
          const int own = (i * GROUPS + group) * 32;
          if (F::kSteps == 1 || key + own < key1)  // not behind the last key
            tile_step<T, D, true, C>(cur + own * B, cur + TILE + own * B, q, key + own, limit,
                                     a.scale2, tile_scales(f, key + own - f.scaled), st, lane);
        }
      wait_loads<0>();
      __syncthreads();
    }
    if (__builtin_expect(st.odd, 0)) {
      for (int k = key0 + max(all_see - key0, 0) / KEYS * KEYS; k < min(key1, limit); ++k) {
        if (((k - key0) / 32) % GROUPS != group) continue;
        const ValueRow<T, D, C> v(a, s, kv, head, k);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const f32x4 x = v.odd_parts(i * 32 + b * 8 + (lane >> 5) * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) st.o[i][4 * b + j] += x[j];
          }
      }
    }
  }

  // Through LDS, which every wave has left: the last barrier above, or no key at all.  The
  // key groups' sums are joined on the way, and rows are written whole.
  constexpr int PITCH = tile_pitch<D>(), HALF = D / 2;
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
  constexpr int STEP = WAVES * 64 / (HALF / 4), BATCH = 4;
  const int first = threadIdx.x / (HALF / 4), d = threadIdx.x % (HALF / 4) * 4;
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
        if (splits == 1) gate[i] = load_gate(a, to[i], side * HALF + d);
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
          write_row<T, D>(a, to[i], side * HALF + d, o, gate[i]);
        } else {
          const int64_t row = ((int64_t)split * a.tokens + to[i].token) * a.q_heads + to[i].head;
          *reinterpret_cast<f32x4 *>(a.tile_part + row * D + side * HALF + d) = o;
        }
      }
    }
  }
}

template <typename T, int D, typename C>
__global__ __launch_bounds__((TileForm<D, C>::kWaves * 64), 2) void attention_tile_kernel(
    Attention a) {
  // One array: with several, the compiler waits for all direct loads at each LDS read.
  __shared__ __attribute__((aligned(16))) char lds[tile_lds<D, C>()];
  tile_rows<T, D, C>(a, blockIdx.x, blockIdx.y, lane_sequence(a), lds);
}

// ------------------------------------------------------------------ both in one launch
// What few rows read more of their keys than 1536 bytes for each key of a tile (in 512 bytes; the mean
// of a sequence's tiles taken for all): few rows come first if it is positive for a call.
template <int D, typename C, int W>
__device__ __forceinline__ int64_t few_lead(const PagedSequence &q, int blocks, int tiles) {
  constexpr int64_t kBlock = kBlockKeys<C, W> * D * Cache<C>::kBytes / 512;
  return blocks * kBlock - (int64_t)tiles * max(q.length - q.count / 2, 0) * 3;
}

// Spans of few rows and places of tiles of a call, for a key-value head, and whether the former come
// first.  All threads of the W waves; sums is free again afterwards.
struct Counts {
  int spans;
  int64_t places;
  bool few_first;
};
template <int D, typename C, int W>
__device__ Counts count_both(const Attention &a, const PagedSequence &mine, uint64_t *sums) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, S = a.batch.sequences;
  TileTotals total = {};
  if (S <= 64) {  // each wave for itself
    const int n = lane < S ? tile_count(a, mine) : 0;
    const int own = lane < S ? few_blocks<C, W>(a, mine) : 0;  // 64 of at most 2^25
    const uint32_t blocks = (uint32_t)__builtin_amdgcn_readlane((int)wave_scan((uint32_t)own), 63);
    if (a.room) total = {(int)wave_total((uint64_t)n), wave_total(all_keys(a, mine, n))};
    const int m = a.room ? tile_places(a, total, mine, n) : 1;
    int64_t lead = 0;
    if (D < 256 && blocks && __any(n > 0))
      lead = (int64_t)wave_total((uint64_t)few_lead<D, C, W>(mine, own, n));
    return {(int)min((uint32_t)a.shares, blocks), (int64_t)wave_total((uint64_t)n * m), lead > 0};
  }
  auto all = [&](uint64_t v) {
    v = wave_total(v);
    __syncthreads();
    if (lane == 0) sums[wave] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < W; ++w) v += sums[w];
    return v;
  };
  uint64_t blocks = 0, tiles = 0, keys = 0, places = 0, lead = 0;
  for (int c = tid; c < S; c += W * 64) {
    const PagedSequence q = paged_sequences(a.batch, c, a.tokens);
    const int n = tile_count(a, q), own = few_blocks<C, W>(a, q);
    blocks += own, tiles += n, keys += all_keys(a, q, n);
    if (D < 256) lead += few_lead<D, C, W>(q, own, n);
  }
  // of a thread's blocks no more than the spans count: both sums in one word
  tiles = all(min(blocks, (uint64_t)a.shares) << 40 | tiles);
  blocks = tiles >> 40, places = tiles &= (1ULL << 40) - 1;
  if (D < 256 && blocks && tiles) lead = all(lead);
  if (a.room) {
    total = {(int)tiles, all(keys)};
    places = 0;
    for (int c = tid; c < S; c += W * 64) {
      const PagedSequence q = paged_sequences(a.batch, c, a.tokens);
      const int n = tile_count(a, q);
      places += (uint64_t)n * tile_places(a, total, q, n);
    }
    places = all(places);
  }
  __syncthreads();
  return {(int)min((uint64_t)a.shares, blocks), (int64_t)places, places && (int64_t)lead > 0};
}

// Workgroups of tiles and of few rows, kTurn of each in turn while there are both: the first bound
// by the matrix cores and a chain of steps, the others by the cache's bytes.  Against a launch each,
// 12 sequences of up to 700 new tokens (heads of 128) take 39 us instead of 45, 2048 tokens behind
// 8192 keys beside 32 of one 263 instead of 310 (64) and 380 instead of 463 (128), 24 of 2 to 24
// 41 instead of 51 (64).  All of one kind first was better for some and 10 % worse than two
// launches for others, as were places for the most that a call can have of each: those without
// work then come before some with it.
// Only where few rows read far more than the tiles do (few_lead) all of them come first: in turn,
// tiles hold places that the last spans wait for, which alone do not keep the memory busy.  64 of one
// behind 1000 to 12000 keys beside short prompts with 1/32 of their keys (heads of 128) 324 us instead
// of 377 and of 333 in two launches, 200 beside 8 prompts 233 instead of 260 and 236, with heads of 64
// 221 instead of 247 and 224.  With 1/4 of the keys both orders took the same (128) or in turn 10 % less
// (64); 100 beside three prompts behind up to 5000 keys 187 instead of 223.  Not with heads of 256,
// where a workgroup has a CU to itself: one behind 200000 keys beside a prompt 63 instead of 56.
// Heads of 128 have a ring of one step here, so that three workgroups still share a CU.  With heads
// of 256 few rows have eight waves as tiles do, one workgroup a CU; of 8 bits 24 sequences of 2 to 24
// tokens take 56 us instead of 63, 64 of one beside two prompts 74 instead of 80, 16 prompts alone
// 75.5 instead of 73.5, two of 1000 tokens (one behind 8000 keys) 254 instead of 245.  Of 16 bits the
// two do not fit the registers there, and have two launches.
template <int D, typename C>
constexpr bool kBoth = D < 256 || Cache<C>::kScaled;
constexpr int kTurn = 256;

template <typename T, int D, typename C>
__global__ __launch_bounds__((TileForm<D, C>::kWaves * 64),
                             (D == 64 ? 4 : D == 128 ? 3 : 2)) void attention_both_kernel(Attention a) {
  constexpr int STEPS = D == 64 ? 2 : 1, W = TileForm<D, C>::kWaves;
  constexpr int FEW = few_lds<D, STEPS, W>(), TILE = tile_lds<D, C>();
  // One array: with several, the compiler waits for all direct loads at each LDS read.
  __shared__ __attribute__((aligned(16))) char lds[FEW > TILE ? FEW : TILE];
  const PagedSequence mine = lane_sequence(a);
  const Counts n = count_both<D, C, W>(a, mine, reinterpret_cast<uint64_t *>(lds));
  const int few = n.spans * a.batch.kv_heads;
  const int64_t tiles = n.places * a.batch.kv_heads;
  // the same for every lane, which the compiler cannot tell of what went through LDS
  const int turns = __builtin_amdgcn_readfirstlane(
      (int)min((int64_t)(few + kTurn - 1) / kTurn, (tiles + kTurn - 1) / kTurn));
  int turn = blockIdx.x / kTurn;
  bool tile = turn < 2 * turns ? turn % 2 == 0 : tiles > few;
  if (__builtin_amdgcn_readfirstlane(n.few_first)) {
    const int own = (few + kTurn - 1) / kTurn;
    tile = turn >= own;
    turn -= tile ? own : 0;
  } else {
    turn = turn < 2 * turns ? turn / 2 : turn - turns;
  }
  const int index = turn * kTurn + blockIdx.x % kTurn;
  const int work = __builtin_amdgcn_readfirstlane(index >= (tile ? tiles : few) ? 0 : tile ? 2 : 1);
  if (work == 2) {
    tile_rows<T, D, C>(a, index, 0, mine, lds);
  } else if (work == 1) {
    few_span<T, D, C, STEPS, W>(a, index, mine, lds);
  }
}

// Rows of sequences in tiles, where their keys were split: D / 4 threads a row, `chunks`
// workgroups a token.
template <typename T, int D>
__device__ __forceinline__ void combine_tile(const Attention &a, int block, int chunks) {
  const int t = block / chunks, lane = threadIdx.x & 63;
  const int i = block % chunks * 256 + threadIdx.x;
  const int head = i / (D / 4), d = i % (D / 4) * 4;
  const int64_t rows = (int64_t)a.tokens * a.q_heads;
  const int64_t row = (int64_t)t * a.q_heads + min(head, a.q_heads - 1);
  // The token's sequence, of which a lane looks at one of 64, and the parts of its row are looked up
  // together; left to itself, the compiler has a round of loads for each.
  int parts = a.room ? a.row_parts[row] : a.splits, lo = 0, hi = 0;
  for (int c = 0; c < a.batch.sequences; c += 64) {
    const int k = min(c + lane, a.batch.sequences - 1);
    int from = a.batch.starts[k], to = a.batch.starts[k + 1];
    asm volatile("" : "+v"(from), "+v"(to), "+v"(parts));
    const uint64_t hit = __ballot(c + lane < a.batch.sequences && from <= t && t < to);
    if (hit) {
      const int at = __builtin_ctzll(hit);
      lo = __builtin_amdgcn_readlane(from, at), hi = __builtin_amdgcn_readlane(to, at);
      break;
    }
  }
  if (lo == hi || head >= a.q_heads) return;  // of no sequence
  const PagedSequence seq = paged_sequence(a.batch, lo, hi, 0, a.tokens);
  if (t >= seq.first + seq.count || (a.few && few_rows(seq, a.group))) return;
  parts = min(parts, a.splits);
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
                             int64_t head_dim, int64_t max_new, int64_t max_keys,
                             bool e4m3 = false) {
  AttentionPlan p = {};
  const int64_t group = q_heads / kv_heads;
  max_new = max_new < tokens ? max_new : tokens;
  p.tile = max_new * group > kFewRows;
  p.few = group <= kFewRows && !(p.tile && sequences == 1);  // one sequence: one of them
  if (p.few) {
    // workgroups that run at a time
    const int64_t all = head_dim == 64 ? 768 : head_dim == 256 && p.tile && e4m3 ? 256 : 512;
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

// Workgroups of attention_combine_kernel for a sequence's key-value head.  Where there are few
// sequences, their rows and channels fill the chip.  Against twice as many workgroups at most, 24
// sequences with 2 to 9 rows took 24.1 instead of 25.2 us and 16 of up to 300 new tokens 34.3 instead
// of 35.6; with half as many, 24 of 2 to 24 (heads of 256), of which three are split in many parts,
// took 69.0 instead of 63.5.
int64_t pair_groups(const AttentionPlan &p, int64_t group, int64_t head_dim) {
  const int64_t units = kFewRows / group * group * (head_dim / 64), some = 2048 / p.parts;
  return some < 1 ? 1 : some < units ? some : units;
}
// And for a token's rows in tiles.
int row_chunks(int64_t q_heads, int64_t head_dim) {
  return (int)((q_heads * (head_dim / 4) + 255) / 256);
}
// Workgroups of attention_both_kernel.
int64_t both_groups(const AttentionPlan &p, int64_t kv_heads) {
  const int64_t tiles = p.tiles * kv_heads * p.splits;
  return ((tiles + kTurn - 1) / kTurn + (p.few_grid + kTurn - 1) / kTurn) * kTurn;
}
// Whether a call's largest launches have fewer than 2^32 threads: of tiles, of sequences' key-value
// heads, of both kinds together, and of the joining of both.
template <bool E4M3_CACHE>
bool attention_fits(const AttentionPlan &p, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                    int64_t head_dim) {
  constexpr int64_t kThreads = 1LL << 32;
  if (p.tiles * kv_heads * 512 >= kThreads) return false;
  if (p.few && p.tile && (head_dim < 256 || E4M3_CACHE) &&
      both_groups(p, kv_heads) * (head_dim == 256 ? 512 : 256) >= kThreads)
    return false;
  const int64_t few = p.few ? p.parts * pair_groups(p, q_heads / kv_heads, head_dim) : 0;
  const int64_t tile = p.splits > 1 ? tokens * row_chunks(q_heads, head_dim) : 0;
  return (few + tile) * 256 < kThreads;
}

template <typename T, int D, typename C>
int launch_attention(const AttentionPlan &p, Attention a, float *workspace, hipStream_t st) {
  a.few = p.few;
  a.part = workspace, a.part_ml = workspace + p.few_rows * D;
  a.tile_part = workspace + p.few_rows * (D + 2), a.tile_ml = a.tile_part + p.tile_rows * D;
  a.parts = reinterpret_cast<Parts *>(a.tile_ml + p.tile_rows * 2);
  a.row_parts = reinterpret_cast<int *>(a.parts + p.parts);
  a.shares = (int)p.shares, a.splits = (int)p.splits, a.room = (int)p.room;
  int64_t ys = 0, tile = 0;  // workgroups that join parts: ys for each of p.parts, and tile
  constexpr bool CAN = kBoth<D, C>;
  const bool both = CAN && p.few && p.tile;
  if (p.few) {
    if (!both) {
      attention_few_kernel<T, D, C><<<(unsigned)p.few_grid, 256, 0, st>>>(a);
      if (const int rc = check_launch("attention_few_kernel")) return rc;
    }
    ys = pair_groups(p, a.group, D);
  }
  const int chunks = row_chunks(a.q_heads, D);
  if (p.tile) {
    const int64_t all = p.tiles * a.batch.kv_heads;
    const dim3 grid((unsigned)(p.room ? all * p.splits : all), (unsigned)(p.room ? 1 : p.splits));
    if (!both) {
      attention_tile_kernel<T, D, C><<<grid, TileForm<D, C>::kWaves * 64, 0, st>>>(a);
      if (const int rc = check_launch("attention_tile_kernel")) return rc;
    } else if constexpr (CAN) {  // of several sequences, whose parts have no dimension of the grid
      attention_both_kernel<T, D, C>
          <<<(unsigned)both_groups(p, a.batch.kv_heads), TileForm<D, C>::kWaves * 64, 0, st>>>(a);
      if (const int rc = check_launch("attention_both_kernel")) return rc;
    }
    if (p.splits > 1) tile = (int64_t)a.tokens * chunks;
  }
  const int64_t all = p.parts * ys + tile;
  if (all == 0) return LM_OK;
  attention_combine_kernel<T, D><<<(unsigned)all, 256, 0, st>>>(a, (int)p.parts, (int)ys, chunks);
  return check_launch("attention_combine_kernel");
}

template <typename T, typename C>
int launch_attention(const AttentionPlan &p, const Attention &a, float *workspace, int head_dim,
                     hipStream_t st) {
  return head_dim == 256   ? launch_attention<T, 256, C>(p, a, workspace, st)
         : head_dim == 128 ? launch_attention<T, 128, C>(p, a, workspace, st)
                           : launch_attention<T, 64, C>(p, a, workspace, st);
}

// The entry points' work: a cache of the rows' type, or of 8 bits with `scales`.
template <bool E4M3_CACHE>
int paged_attention(const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads,
                    const void *k_pages, const void *v_pages, const float *scales,
                    int64_t scale_stride, int64_t pages, int64_t page_stride, int64_t kv_heads,
                    int64_t page_size, int64_t head_dim, const int32_t *starts,
                    const int32_t *lengths, const int32_t *table, int64_t table_stride,
                    int64_t table_pages, int64_t sequences, int64_t tokens, int64_t max_new,
                    float scale, const void *gate, int64_t gate_token_stride,
                    int64_t gate_head_stride, void *out, void *workspace, int64_t workspace_bytes,
                    int dtype, void *stream) {
  if (const int rc = paged_check(pages, page_stride, kv_heads, page_size, head_dim, starts, lengths,
                                 table, table_stride, table_pages, sequences, tokens, dtype))
    return rc;
  if (E4M3_CACHE)
    if (const int rc = scales_check(scales, scale_stride, kv_heads, page_size, page_stride,
                                    tokens == 0 || sequences == 0))
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
                                            table_pages * page_size, E4M3_CACHE);
  LM_REQUIRE(sequences * kv_heads < (1LL << 24) &&
                 attention_fits<E4M3_CACHE>(plan, tokens, q_heads, kv_heads, head_dim),
             LM_EINVAL, "too many rows");
  const int64_t need = attention_bytes(plan, head_dim);
  LM_REQUIRE(need == 0 || (workspace && aligned16(workspace)), LM_EINVAL,
             "attention needs a 16-byte aligned workspace");
  LM_REQUIRE(workspace_bytes >= need, LM_ENOMEM, "the workspace is too small");
  Attention a = {};
  a.q = static_cast<const uint16_t *>(q), a.q_token = q_token_stride, a.q_head = q_head_stride;
  a.gate = static_cast<const uint16_t *>(gate);
  a.gate_token = gate_token_stride, a.gate_head = gate_head_stride;
  a.k_pages = k_pages, a.v_pages = v_pages;
  a.scales = scales, a.scale_stride = scale_stride;
  a.out = static_cast<uint16_t *>(out);
  a.batch = {starts, lengths, table, table_stride, (int)sequences, (int)table_pages,
             __builtin_ctzll((unsigned long long)page_size), (int)pages, page_stride,
             (int)kv_heads};
  a.tokens = (int)tokens, a.q_heads = (int)q_heads, a.group = (int)(q_heads / kv_heads);
  // A scale of 0 as one too small to matter, so that a masked -inf stays one under it.
  a.scale2 = fmaxf(scale2, 1e-30f);
  a.flip = scale < 0.0f ? 0x80008000u : 0u;
  float *ws = static_cast<float *>(workspace);
  using CB = std::conditional_t<E4M3_CACHE, E4M3, BF16>;
  using CF = std::conditional_t<E4M3_CACHE, E4M3, FP16>;
  return dtype == LM_BF16
             ? launch_attention<BF16, CB>(plan, a, ws, (int)head_dim, as_stream(stream))
             : launch_attention<FP16, CF>(plan, a, ws, (int)head_dim, as_stream(stream));
}

}  // namespace
}  // namespace lm
