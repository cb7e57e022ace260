// What the kernels over a paged cache share: which sequence a token belongs to, where a position
// of it is stored.
#pragma once
#include "elem_types.h"

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, "Division by invariant
// integers using multiplication").
struct FastDiv {
  uint32_t d, mul, shift;
  FastDiv() = default;
  explicit FastDiv(uint32_t divisor) : d(divisor), shift(0) {
    while ((1ull << shift) < divisor) ++shift;
    mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - divisor)) / divisor + 1);
  }
  QMOE_HOST_DEV uint32_t div(uint32_t n) const { return (uint32_t)((((uint64_t)n * mul) >> 32) + n) >> shift; }
};

// Positions that a table can name (so that those of whole tiles beyond them are ints too).
constexpr long TOKENS_MAX = 0x7ffff000l;

// A cache tensor [pages, page, heads, D] as element steps; elements of a head are contiguous.
struct CacheSteps {
  long page, slot, head;
};

// The batch: `starts` [B + 1] (rows [starts[b], starts[b + 1]) of the new tokens are sequence b's; null: row
// b is), `lengths` [B] (with the new tokens), `table` [B, width] of pages.
struct Batch {
  const int *table, *lengths, *starts;
  long table_ld, n_pages;
  int T, B, width;
  FastDiv page;

  // Sequence of row t (wave-uniform; every lane calls): how many sequences end at or before t; B
  // behind the last one.
  QMOE_DEV int sequence(int t) const {
    if (!starts) return t;
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int i = 0; i < B; i += 64) b += __popcll(__ballot(i + lane < B && starts[i + lane + 1] <= t));
    return b;
  }
  // First new row and number of new rows of sequence b; both within [0, T] whatever `starts` holds.
  QMOE_DEV int start(int b) const { return starts ? min(max(starts[b], 0), T) : b; }
  QMOE_DEV int first_row(int b) const { return start(b); }
  QMOE_DEV int new_rows(int b) const { return starts ? max(start(b + 1) - start(b), 0) : 1; }
  // Cached tokens of sequence b, as many as its row of the table can hold.
  QMOE_DEV int length(int b) const {
    const long most = n_pages ? (long)width * page.d : 0;
    return (int)min(max((long)lengths[b], 0l), most);
  }
  // The page of position p in [0, length(b)), or -1 where the table names none of the cache's.
  QMOE_DEV long page_of(int b, int p) const {
    const int e = table[b * table_ld + page.div(p)];
    return e >= 0 && e < n_pages ? e : -1;
  }
};

// Whether a call lacks a tensor that has elements.
static inline bool missing(const void* k_cache, const void* v_cache, long n_pages, const void* table, int width,
                           const void* lengths, int B) {
  return (n_pages && (!k_cache || !v_cache)) || (B && (!lengths || (width && !table)));
}
