// How attention over rows that share pages is dealt out (csrc/paged_shared_attention.cu): plain C++, used by the kernels, their launcher and
// (through the host simulator library) by the CPU tests.
//
// An element is what some rows see in common: the shared positions of a group of rows, or the own positions of one row.  Its items are
// a KV head each, and `kQueries` of the (row, query head) pairs that go with it.  An item is some units for its start and two for every tile
// of positions, three for one that meets two tiles of queries.  All items lie in a line, cut into equal shares, a CTA each; a piece is what a CTA has of an item.  The kernel that
// joins the pieces finds them from the line alone.
#pragma once
#include "paged_plan.h"

namespace penny {
namespace paged {

// kItemStart: an item's start and end (queries in, part of the output out).  kLeastUnits: of a CTA.  (A tile of two times 128 queries 4200
// clocks, one of up to 128 2600, an item 1300 more: 100 rows of 16000 shared positions and 500 each 118 us with all tiles alike, so 101.)
constexpr int kItemStart = 1, kTileUnits = 2, kPairUnits = 3, kLeastUnits = 3;
constexpr long long kMaxSharedUnits = 1ll << 30;

PENNY_ATTN_HD int tiles_of(int positions, int tile) { return positions > 0 ? (positions - 1) / tile + 1 : 0; }
PENNY_ATTN_HD int item_units(int tiles, bool pair) { return tiles > 0 ? kItemStart + tiles * (pair ? kPairUnits : kTileUnits) : 0; }
PENNY_ATTN_HD int unit_share(int units, int ctas) { return attn::at_least(kLeastUnits, (units - 1) / ctas + 1); }
// The tiles that CTA `cta` has of an item whose first unit is `begin`: those whose first unit is in its share.
struct Tiles {
  int from, to;
};
PENNY_ATTN_HD int first_tile(long long unit, int tiles, bool pair) {  // the first that begins at `unit` of the item's tiles or behind it
  const int each = pair ? kPairUnits : kTileUnits;
  return unit <= 0 ? 0 : unit > (long long)tiles * each ? tiles : (int)((unit + each - 1) / each);
}
PENNY_ATTN_HD Tiles piece_of(int begin, int tiles, bool pair, int share, int cta) {
  const long long from = (long long)cta * share - begin - kItemStart;
  return {first_tile(from, tiles, pair), first_tile(from + share, tiles, pair)};
}
PENNY_ATTN_HD int cta_of(int begin, int tile, bool pair, int share) { return (begin + kItemStart + tile * (pair ? kPairUnits : kTileUnits)) / share; }
// Whether a batch whose rows can see `positions` each is worth the shared kernel's tiles.  The one that reads every row by itself finds what they
// share in L2, and needs no time to start tensor cores: us with / without, of bytes for all rows, 32 of 8 heads of 128: 138 MB 25 / 20, 167 30 /
// 22, 543 36 / 49, 554 38 / 51, 2174 48 / 165; e4m3 272 MB 41 / 39 and 44 / 41, 1087 55 / 131; 20 of 20 of 64, fp16: 170 MB 29 / 24, 173 21 / 25, 209 30 / 28,
// 679 31 / 71; 4 of 1: 272 MB 51 / 30.  (The lengths are on the device; a table's width says what they can be.)
inline bool shared_pays(long long rows, long long positions, int kv_heads, int dim, int value_bytes) {
  return rows * positions * kv_heads * dim * 2 * value_bytes > 256ll << 20;
}
// A row takes what its group shares, the group's first `shared` positions, if it sees all of it; one whose window leaves some out, or that was cut
// back since, reads what it sees by itself.  (A weight of zero does not take a value that is not finite out of a product.)
PENNY_ATTN_HD bool takes_part(const Seen& seen, int shared) { return seen.first == 0 && shared <= seen.end; }
// What of `shared` positions is worth reading for a group: nothing where a row that has them all cannot see them all, else all that a table can
// hold.  (Of a row that sees nothing else the window may end with them.)
PENNY_ATTN_HD int group_end(int shared, int max_len, int window) {
  const int end = attn::cached_rows(shared, max_len);
  return window > 0 && end > window ? 0 : end;
}
// (row, query head) pairs of an item, and of how many items: of `queries` pairs, `most` to an item
PENNY_ATTN_HD int query_tiles(int queries, int most) { return (queries + most - 1) / most; }
// The items of an element are alike but for its last queries of each head, which may be fewer; they count as the others do.
PENNY_ATTN_HD bool pair_of(int queries, int most) { return most > 128 && queries > 128; }
// Units of a batch at most, if every row sees `positions`: shared and own ones of every row, each by itself.
inline long long most_units(long long rows, int kv_heads, int group, long long positions, int tile, int most) {
  return 2 * rows * kv_heads * ((group + most - 1) / most) * (kItemStart + kPairUnits * ((positions + tile - 1) / tile));
}

// Tiles of a head size: positions, and (row, query head) pairs that an item takes at most (tensor memory and shared memory hold two tiles of 128
// queries for heads of up to 128, one for 256).
PENNY_ATTN_HD constexpr int tile_positions(int dim) { return dim <= 128 ? 128 : 64; }
PENNY_ATTN_HD constexpr int tile_queries(int dim) { return dim <= 128 ? 256 : 128; }
// Whether the line of a batch whose tables hold `positions` a row can be counted, and its heads be a grid's; others are read each row by itself.
inline bool shared_fits(long long rows, int kv_heads, int group, long long positions, int dim) {
  return kv_heads <= 65535 && most_units(rows, kv_heads, group, positions, tile_positions(dim), tile_queries(dim)) <= kMaxSharedUnits;
}

}  // namespace paged
}  // namespace penny
