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

// Where a slot lies, in units of the steps, if it is one of the pool's; -1 if not.  (Slots and tables are the caller's memory on the
// device: what they say is looked at, never trusted.)
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

// How a batch is shared out.  A row's (KV head, head group) pairs are its items; a team is one CTA for each item, so that a page's
// heads are read at about the same time (apart from each other 64 rows of 16000 positions, e4m3, took 389 us instead of 340).  The
// rows lie in a line, each kStart units for its start (q on the way in, the output) and one for every tile of positions, an empty
// one a single unit; every warp of a team's CTAs gets `share` units, at least kMinShare (4 / 5 / 6: 3 rows of 300 positions 8.2 / 8.9 /
// 9.7 us).  The lengths are on the device, and every warp sums over them by itself.
// kStart: 96 rows of 1 to 8192 positions, e4m3, in 49.3 / 45.4 / 43.9 / 43.0 us with 1 / 2 / 3 / 5; 256 of 100 25.5 / 27.3 / 27.0 / 25.0.
constexpr int kMinShare = 4, kStart = 3;
constexpr long long kMaxLen = 0x7fff0000, kMaxUnits = 1ll << 30;  // (all rows' units, and a share more, fit 32 bits)

PENNY_ATTN_HD int units_of(int positions, int tile) { return positions > 0 ? kStart + (positions + tile - 1) / tile : 1; }
PENNY_ATTN_HD int share_of(int units, int warps) { return attn::at_least(kMinShare, (int)(((uint32_t)units + warps - 1) / (uint32_t)warps)); }
// Teams of a launch: as many as the GPU holds (`slots` CTAs), in more rounds where that leaves over a tenth of it empty; no more
// than there are shares of tiles, if every row has `units` units.
inline int teams_of(long long rows, int items, long long units, int warps, int slots) {
  int best = 1;
  double used = 0;
  for (int rounds = 1; rounds <= 8 && used < 0.9; ++rounds) {
    const int teams = slots * rounds / items;
    const double now = (double)teams * items / ((double)slots * rounds);
    if (teams > 0 && now > used) best = teams, used = now;
  }
  const long long most = (rows * (units - kStart) + (long long)warps * kMinShare - 1) / ((long long)warps * kMinShare);
  return most < best ? (int)(most > 1 ? most : 1) : best;
}

// What a warp has of the line: where it stands in a row, and what is left of its share.
struct Walk {
  int row;
  int at, units;   // units of the row that lie behind, and all of them
  int first, end;  // positions
  int left;        // units of the share
};
// A part of a row: its tiles [from, to); begins and ends: the row does.
struct WalkPart {
  int from, to;
  bool begins, ends;
};
template <class SeenOf>  // SeenOf(row): what a row attends to
PENNY_ATTN_HD void enter_row(Walk& w, int tile, SeenOf seen) {
  const Seen s = seen(w.row);
  w.first = s.first;
  w.end = s.end;
  w.units = units_of(s.end - s.first, tile);
}
// The next part of the share (w.left > 0): all that it has of one row.  Without tiles: an empty row (which begins and ends), or a
// row's start alone, which is nothing (the next warp's part begins the row).
template <class SeenOf>
PENNY_ATTN_HD WalkPart next_part(Walk& w, int tile, SeenOf seen) {
  if (w.at == w.units) {
    ++w.row;
    w.at = 0;
    enter_row(w, tile, seen);
  }
  const int from = attn::at_least(0, w.at - kStart), end = attn::at_most(w.units, w.at + w.left), to = attn::at_least(0, end - kStart);
  w.left -= end - w.at;
  w.at = end;
  const bool some = to > from || w.first == w.end;
  return {from, to, from == 0 && some, end == w.units && some};
}
// What lies across the end of a team's share, [begin, end) of the line: the row that has unit `end` starts at unit `start`.  How many
// teams behind it have a part of the row, if its first tile is the team's; 0: the row is another team's.
PENNY_ATTN_HD int teams_behind(int begin, int end, int start, int units) {
  const int first = start + kStart, behind = start + units - end, each = end - begin;
  return first >= begin && first < end && behind > 0 ? (behind + each - 1) / each : 0;
}

// A pool's strides in a unit so large that a place in it fits 32 bits: the largest power of two that divides both.  bytes 0:
// no such unit (more than 2^32 - 1 times what divides the strides).
struct Steps {
  uint32_t page, pos, bytes;
};
inline Steps steps_of(long long pages, long long page_size, long long page_stride, long long pos_stride, int value_bytes) {
  long long page = page_stride * value_bytes, pos = pos_stride * value_bytes;
  uint32_t bytes = 1;
  // (the strides of a single page or position say nothing)
  if (pages == 1) page = 0;
  if (page_size == 1) pos = 0;
  while (bytes < (1u << 30) && ((page | pos) & 1) == 0 && (page | pos) != 0) page >>= 1, pos >>= 1, bytes <<= 1;
  const long long limit = 0xffffffffll;
  if (page > limit || pos > limit || (pages - 1) * page > limit || (page_size - 1) * pos > limit || (pages - 1) * page + (page_size - 1) * pos >= limit)
    return {0, 0, 0};
  return {(uint32_t)page, (uint32_t)pos, bytes};
}
constexpr uint32_t kNoStep = 0xffffffffu;
// Where position `pos` lies, in such units, if its page is one of the pool's; kNoStep if not.
PENNY_ATTN_HD uint32_t step_of(int page, int pages, int pos, const PageDiv& d, uint32_t page_step, uint32_t pos_step) {
  return (uint32_t)page < (uint32_t)pages ? (uint32_t)page * page_step + (uint32_t)(pos - div_page(d, pos) * (int)d.size) * pos_step : kNoStep;
}

}  // namespace paged
}  // namespace penny
