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
// share in L2, and needs no time to start tensor cores.  What decides is how much the rows hold and share, which only the device knows;
// by what they can hold, the shared kernel's time over the other's (16 / 64 / 200 rows full of positions, 94 % of them shared; `-`: not timed):
//   heads                 275 MB             350                430                520                620                800                1100
//   32 of 8 of 128 bf16   1.05 1.23 1.95     0.92 1.07 1.65     0.86 0.92 1.45     0.77 0.82 1.29     0.72 0.83 1.03     0.65 0.69 0.94     0.59 0.60 0.75
//   the same e4m3         1.16 1.30 1.86     1.01 1.13 1.56     0.93 0.96 1.35     0.87 0.86 1.16     0.81 0.82 0.93     0.78 0.67 1.04     0.69 0.58 0.84
//   4 of 1 of 128 bf16    2.39 1.29 1.22     2.06 1.15 1.08     1.81 1.04 0.99     1.62 0.97 0.86     -    0.85 0.84     -    0.73 0.68     -    0.62 0.58
//   28 of 2 of 128 e4m3   2.46 1.77 1.39     1.91 1.51 1.14     1.78 1.40 1.10     1.63 1.25 0.97     -    1.11 0.89     -    1.01 0.82     -    0.81 0.69
//   8 of 1 of 256 bf16    2.87 1.42 1.29     2.51 1.31 1.14     2.22 1.18 1.03     2.01 1.08 0.95     1.73 0.98 0.87     1.49 0.85 0.75     1.20 0.74 0.67
//   20 of 20 of 64 fp16   0.82 0.92 -        0.77 0.79 2.23     0.68 0.69 1.77     0.65 0.59 1.58     0.58 0.51 1.33     0.54 0.56 1.07     0.50 0.45 0.81
// With 80 % shared 0.8 to 1.4 at 1100 MB, with 30 % 1.1 to 3.1 at any size: a row's own positions take longer here, so such rows go without groups.
inline bool shared_pays(long long rows, long long positions, int kv_heads, int dim, int value_bytes) {
  return (double)rows * positions * kv_heads * dim * 2 * value_bytes > 512ll << 20;  // (heads of stride zero: more than 64 bits hold)
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
