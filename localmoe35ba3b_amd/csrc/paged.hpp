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

__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch &b, int s, int tokens) {
  const int lo = b.starts[s], hi = b.starts[s + 1], len = b.lengths[s];
  const int room = b.table_pages << b.page_shift;
  const int first = min(max(lo, 0), tokens);
  return {first, max(min(hi, tokens) - first, 0), len - (hi - lo) + (first - lo),
          min(max(len, 0), room)};
}

// Element offset of position p's page of sequence s.
__device__ __forceinline__ int64_t paged_page(const PagedBatch &b, int s, int p) {
  const int i = min(p >> b.page_shift, b.table_pages - 1);
  return clamp_index32(b.table[s * b.table_stride + i], b.pages) * b.page_stride;
}

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

}  // namespace lm
