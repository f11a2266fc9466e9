// A batch of sequences over a paged cache, as the attention operators read it:
// sequence s's new tokens are the rows starts[s] .. starts[s + 1] - 1 of the
// call's inputs and the last of its lengths[s] positions; position p lives in
// row p % page_size of page table[s][p / page_size].  A page holds
// [kv_heads][page_size][head_dim] values.
//
// Every value read from the arrays is clamped before it becomes an address, so
// malformed ones give wrong values, never an access outside the buffers.
#pragma once

#include "internal.hpp"

namespace lm {

struct PagedBatch {
  const int32_t *starts, *lengths, *table;
  int64_t table_stride;  // between sequences
  int sequences, table_pages;
  int page_shift;  // page_size = 1 << page_shift
  int pages;
  int64_t page_stride;  // elements between pages
  int kv_heads;
};

// One sequence's share of a call: row first + i is position base + i and sees the
// positions up to its own, none from length on.
struct PagedSequence {
  int first, count, base, length;
};

__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch &b, int lo, int hi, int len,
                                                       int tokens) {
  const int room = b.table_pages << b.page_shift;
  const int first = min(max(lo, 0), tokens);
  return {first, max(min(hi, tokens) - first, 0), len - (hi - lo) + (first - lo),
          min(max(len, 0), room)};
}

__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch &b, int s, int tokens) {
  return paged_sequence(b, b.starts[s], b.starts[s + 1], b.lengths[s], tokens);
}
// Sums over the lanes up to each of a wave (whole numbers), without the LDS round trips of shuffles:
// within 16 lanes, then over the 16s and the halves before.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lanes_before(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t lanes_before(uint64_t v) {
  return (uint64_t)lanes_before<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 |
         lanes_before<CTRL, ROWS>((uint32_t)v);
}
template <typename U>
__device__ __forceinline__ U wave_scan(U v) {
  v += lanes_before<0x111, 0xF>(v);
  v += lanes_before<0x112, 0xF>(v);
  v += lanes_before<0x114, 0xF>(v);
  v += lanes_before<0x118, 0xF>(v);
  v += lanes_before<0x142, 0xA>(v);  // lane 15 of the 16 before
  v += lanes_before<0x143, 0xC>(v);  // lane 31
  return v;
}
__device__ __forceinline__ uint64_t wave_total(uint64_t v) {
  const uint64_t s = wave_scan(v);
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(s >> 32), 63) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)s, 63);
}

// The sequence of each lane, looked up in one round of loads: left to itself, the compiler looks for
// the length only where the starts leave new tokens.
__device__ __forceinline__ PagedSequence paged_sequences(const PagedBatch &b, int s, int tokens) {
  int lo = b.starts[s], hi = b.starts[s + 1], len = b.lengths[s];
  asm volatile("" : "+v"(lo), "+v"(hi), "+v"(len));
  return paged_sequence(b, lo, hi, len, tokens);
}
// Sequence s, the same for every lane: of up to 64 from the lane that has it.
__device__ __forceinline__ PagedSequence sequence_at(const PagedBatch &b, int s,
                                                     const PagedSequence &mine, int tokens) {
  if (b.sequences <= 64)
    return {__builtin_amdgcn_readlane(mine.first, s), __builtin_amdgcn_readlane(mine.count, s),
            __builtin_amdgcn_readlane(mine.base, s), __builtin_amdgcn_readlane(mine.length, s)};
  const PagedSequence q = paged_sequences(b, s, tokens);
  return {__builtin_amdgcn_readfirstlane(q.first), __builtin_amdgcn_readfirstlane(q.count),
          __builtin_amdgcn_readfirstlane(q.base), __builtin_amdgcn_readfirstlane(q.length)};
}

// Position p's page of sequence s, and its element offset.
__device__ __forceinline__ int paged_number(const PagedBatch &b, int s, int p) {
  const int i = min(p >> b.page_shift, b.table_pages - 1);
  return clamp_index32(b.table[s * b.table_stride + i], b.pages);
}
__device__ __forceinline__ int64_t paged_page(const PagedBatch &b, int s, int p) {
  return paged_number(b, s, p) * b.page_stride;
}

// A cache in 8 bits holds e4m3 values (four significant bits, up to 448, no infinities) and a
// scale, a power of two, for each kScaleKeys positions of a head, keys and values apart.
struct E4M3 {};
constexpr int kScaleKeys = 16, kScaleShift = 4;
// Exponents of scales for rows of type T: the least keeps steps of 2^-9 of a scale in T, the largest
// a value of four significant bits that T holds, kHeldMost (61440 in fp16).
template <typename T>
constexpr int kScaleLeast = __is_same(T, FP16) ? -15 : -117;
template <typename T>
constexpr int kScaleMost = __is_same(T, FP16) ? 8 : 120;
template <typename T>
constexpr float kHeldMost = __is_same(T, FP16) ? 61440.0f : 0x1.Ep127f;

// A launch has fewer than 2^32 threads; the kernels take at most 256 for a token.
constexpr int64_t kMaxTokens = 1LL << 24;

// Positions are 32 bits in the kernels, which look up to 1024 past the one they are at (the pages
// of the next steps, a tile's last keys).
constexpr int64_t kMaxPositions = (1LL << 31) - 4096;

// Host checks of what the entry points of the paged cache share; LM_OK or the status.
inline int paged_check(int64_t pages, int64_t page_stride, int64_t kv_heads, int64_t page_size,
                       int64_t head_dim, const void *starts, const void *lengths,
                       const void *table, int64_t table_stride, int64_t table_pages,
                       int64_t sequences, int64_t tokens, int dtype) {
  LM_REQUIRE(dtype == LM_BF16 || dtype == LM_FP16, LM_EINVAL, "attention requires FP16/BF16");
  LM_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, LM_EINVAL,
             "attention supports heads of 64, 128 or 256");
  LM_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0, LM_EINVAL,
             "page size must be a power of two from 16 to 1024");
  LM_REQUIRE(kv_heads >= 1 && kv_heads <= 1024, LM_EINVAL, "invalid number of key-value heads");
  LM_REQUIRE(pages >= 1 && pages < (1LL << 31) && page_stride >= kv_heads * page_size * head_dim &&
                 page_stride % 8 == 0,
             LM_EINVAL, "invalid pages");
  LM_REQUIRE(tokens >= 0 && tokens < kMaxTokens, LM_EINVAL, "invalid token count");
  LM_REQUIRE(sequences >= 0 && sequences <= 65536, LM_EINVAL, "invalid number of sequences");
  LM_REQUIRE(table_pages >= 1 && table_pages <= kMaxPositions / page_size && table_stride >= 0,
             LM_EINVAL, "invalid page table");
  LM_REQUIRE(tokens == 0 || sequences == 0 || (starts && lengths && table), LM_EINVAL,
             "null pointer");
  return LM_OK;
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Of a cache in 8 bits: its scales, and pages whose rows stay 16-byte aligned.
inline int scales_check(const float *scales, int64_t scale_stride, int64_t kv_heads,
                        int64_t page_size, int64_t page_stride, bool empty) {
  LM_REQUIRE(page_stride % 16 == 0, LM_EINVAL, "invalid pages");
  LM_REQUIRE(scale_stride >= 2 * kv_heads * (page_size / kScaleKeys), LM_EINVAL,
             "invalid scales of the pages");
  LM_REQUIRE(empty || (scales && (reinterpret_cast<uintptr_t>(scales) & 3) == 0), LM_EINVAL,
             "invalid scales of the pages");
  return LM_OK;
}

}  // namespace lm
