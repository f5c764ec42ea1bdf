// How attention over rows that share pages is dealt out (csrc/paged_shared_attention.cu): plain C++, used by the kernels, their launcher and
// (through the host simulator library) by the CPU tests.
//
// An element is what some rows see in common: the shared positions of a group of rows, or the own positions of one row.  Its items are
// a KV head each, and `kQueries` of the (row, query head) pairs that go with it.  An item is a few units for its start and one for every tile
// of positions.  All items lie in a line, cut into equal shares, a CTA each; a piece is what a CTA has of an item.  The kernel that
// joins the pieces finds them from the line alone.
#pragma once
#include "paged_plan.h"

namespace penny {
namespace paged {

// kItemStart: an item's start and end (queries in, part of the output out) in tiles.  kLeastUnits: of a CTA.
constexpr int kItemStart = 1, kLeastUnits = 2;
constexpr long long kMaxSharedUnits = 1ll << 30;

PENNY_ATTN_HD int tiles_of(int positions, int tile) { return positions > 0 ? (positions - 1) / tile + 1 : 0; }
PENNY_ATTN_HD int item_units(int tiles) { return tiles > 0 ? kItemStart + tiles : 0; }
PENNY_ATTN_HD int unit_share(int units, int ctas) { return attn::at_least(kLeastUnits, (units - 1) / ctas + 1); }
// The tiles that CTA `cta` has of an item whose first unit is `begin`.
struct Tiles {
  int from, to;
};
PENNY_ATTN_HD int inside(long long x, int most) { return x < 0 ? 0 : x > most ? most : (int)x; }
PENNY_ATTN_HD Tiles piece_of(int begin, int tiles, int share, int cta) {
  const long long from = (long long)cta * share - begin - kItemStart;
  return {inside(from, tiles), inside(from + share, tiles)};
}
PENNY_ATTN_HD int cta_of(int begin, int tile, int share) { return (begin + kItemStart + tile) / share; }
// (row, query head) pairs of an item, and of how many items: of `queries` pairs, `most` to an item
PENNY_ATTN_HD int query_tiles(int queries, int most) { return (queries + most - 1) / most; }
// Units of a batch at most, if every row sees `positions`: shared and own ones of every row, each by itself.
inline long long most_units(long long rows, int kv_heads, int group, long long positions, int tile, int most) {
  return 2 * rows * kv_heads * ((group + most - 1) / most) * (kItemStart + (positions + tile - 1) / tile);
}

}  // namespace paged
}  // namespace penny
