// Index arithmetic of the paged KV cache (csrc/paged_*.cu): plain C++, used by the kernels, by their launchers and (through
// the host simulator library) by the CPU tests.
#pragma once
#include <stdint.h>

#include "decode_attn_plan.h"

namespace penny {
namespace paged {

// Division of a position by the page size, any page size: q = n m / 2^(31 + l) with l = ceil(log2 d), m = ceil(2^(31 + l) / d).
// m d exceeds 2^(31 + l) by less than d <= 2^l, so the quotient is exact for n < 2^31 (Granlund and Montgomery, Division by
// invariant integers using multiplication, 1994).
struct PageDiv {
  uint32_t size, mul;
  int shift;
};
inline PageDiv page_div(int size) {
  int l = 0;
  while ((1ll << l) < size) ++l;
  const uint64_t pow = 1ull << (31 + l);
  return {(uint32_t)size, (uint32_t)((pow + size - 1) / size), 31 + l};
}
PENNY_ATTN_HD int div_page(const PageDiv& d, int n) { return (int)(((uint64_t)(uint32_t)n * d.mul) >> d.shift); }
// pages that hold n positions
PENNY_ATTN_HD int pages_of(const PageDiv& d, int n) { return n > 0 ? div_page(d, n - 1) + 1 : 0; }

// Where position `pos` lies, in units of the steps, if its page is one of the pool's; -1 if not.  (A table is the caller's memory on
// the device: what it says is looked at, never trusted.)
PENNY_ATTN_HD long long place_of(int page, int pages, int pos, const PageDiv& d, long long page_step, long long pos_step) {
  return (uint32_t)page < (uint32_t)pages ? page * page_step + (pos - div_page(d, pos) * (int)d.size) * pos_step : -1;
}
// The same for a slot.
PENNY_ATTN_HD long long place_of_slot(long long slot, int pages, int page_size, long long page_step, long long pos_step) {
  if (slot < 0 || slot >= (long long)pages * page_size) return -1;
  const long long page = slot / page_size;
  return page * page_step + (slot - page * page_size) * pos_step;
}

// What a row of `length` positions attends to: [first, end), its last `window` positions (0: all), no more than a table row
// can hold.
struct Seen {
  int first, end;
};
PENNY_ATTN_HD Seen seen_of(int length, int max_len, int window) {
  const int end = attn::cached_rows(length, max_len);
  return {window > 0 && end > window ? end - window : 0, end};
}

// How the rows of a batch are cut: into pieces of `len` positions or a little more, so that all (row, head group) pairs
// together make about `slots` CTAs.  The lengths are on the device; the launcher makes the grid for the most pieces that
// any lengths can ask for, and every CTA counts through the cut by itself.
constexpr int kMinPiece = 256, kMaxPieces = 128;

PENNY_ATTN_HD int piece_len(long long total, int items_per_row, int slots) {
  const long long len = (total * items_per_row + slots - 1) / slots;
  return len < kMinPiece ? kMinPiece : len > 0x7fffffff ? 0x7fffffff : (int)len;
}
PENNY_ATTN_HD int pieces_of(int rows, int len) { return attn::at_most(kMaxPieces, attn::at_least(1, rows / len)); }
// CTAs beyond one per (row, head group): floor(rows / len) summed over the rows is at most total / len, so all pieces of all
// head groups are at most `slots` and one for each pair; no more than the longest row can have either.
inline long long extra_pieces(long long rows, int items_per_row, int slots, int most_seen) {
  const long long by_len = rows * items_per_row * (pieces_of(most_seen, kMinPiece) - 1);
  return by_len < slots ? by_len : slots;
}

}  // namespace paged
}  // namespace penny
