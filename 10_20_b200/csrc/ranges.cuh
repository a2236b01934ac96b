// How a line of tiles lies in equal ranges, one CTA or warp each, and what a join
// learns of it.  Host and device.
//
// The tiles of all rows stand in a line; a row that lies in several ranges is joined
// from the parts that they leave.  Every range records where it begins, and a row is
// joined on behalf of the first range that begins inside it.  With fewer tiles than
// ranges the last ranges are empty and begin where the line ends, in no row: a record
// that named a row all the same would have range 1 cut the line's only tile, whose
// range leaves no part.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define V1X_HD __host__ __device__ __forceinline__
#else
#define V1X_HD inline
#endif

namespace v1x {
namespace attn {

struct RangeBegin {
  int64_t place;   // the row (or the row and its segment) in which the range begins
  int64_t first;   // that row's first tile in the line
  int64_t tiles;   // that row's tiles
  int64_t begin;   // the range's own first tile
};

// The first tile of range x: ranges of `base` units, the first `extra` of them one more.
V1X_HD int64_t range_start(int64_t x, int64_t unit, int64_t base, int64_t extra) {
  return (x * base + (x < extra ? x : extra)) * unit;
}

// The record of a range that begins in no row: no tiles, so it is inside none.
V1X_HD RangeBegin no_row(int64_t begin) { return RangeBegin{0, begin, 0, begin}; }

// The record of the range that begins at tile `begin`, which lies behind the rows before
// `row`; that one's first tile is `first`.
template <typename Tiles>
V1X_HD RangeBegin find_begin(int64_t begin, int64_t row, int64_t rows, int64_t first, Tiles tiles) {
  for (; row < rows; ++row) {
    const int64_t n = tiles(row);
    if (begin < first + n) return RangeBegin{row, first, n, begin};
    first += n;
  }
  return no_row(begin);
}

V1X_HD bool begins_inside(const RangeBegin& r) { return r.begin > r.first && r.begin < r.first + r.tiles; }

// The range is the first one to begin inside its row; `before`: where the range before it begins.
V1X_HD bool cuts_first(const RangeBegin& r, int64_t before) { return begins_inside(r) && before <= r.first; }

// The records of all ranges, four words each, [ranges + 1] of them; of the last one only
// `begin` is there, the number of all tiles.  (As an array of the struct the joins of
// many rows took 72 to 84 registers instead of 60, and 100 rows of 2048 tokens 82 us
// instead of 76.)
V1X_HD void put_record(int64_t* where, int64_t x, const RangeBegin& r) {
  where[4 * x] = r.place;
  where[4 * x + 1] = r.first;
  where[4 * x + 2] = r.tiles;
  where[4 * x + 3] = r.begin;
}
V1X_HD RangeBegin record_of(const int64_t* where, int x) {
  return RangeBegin{where[4 * x], where[4 * x + 1], where[4 * x + 2], where[4 * x + 3]};
}
V1X_HD int64_t begin_of(const int64_t* where, int x) { return where[4 * x + 3]; }

}  // namespace attn
}  // namespace v1x
