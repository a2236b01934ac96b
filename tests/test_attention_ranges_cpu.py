"""CPU: which rows the attention kernels join, from the host side of csrc/ranges.cuh.

A program built from the header lays random batches of short rows out in ranges as
the kernels do (every range finds its own beginning), and lets the joins choose: with
one warp a part by the record of each range, with sixteen by a search for the row.  A
row that lies in several ranges that are not empty has to be joined once, from exactly
those ranges' parts; no other row may be touched."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "10_20_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <algorithm>
#include <map>
#include <vector>

#include "ranges.cuh"

using namespace v1x::attn;

static unsigned long long seed = 12345;
static int64_t draw(int64_t n) {   // 0 .. n - 1
  seed = seed * 6364136223846793005ull + 1442695040888963407ull;
  return static_cast<int64_t>((seed >> 33) % n);
}

// segments: of a row, each of the row's tiles (1: the row itself)
static int batch(const std::vector<int64_t>& tiles, int64_t segments, int64_t ranges, const char* what) {
  const int64_t rows = tiles.size();
  int64_t all = 0;
  for (int64_t t : tiles) all += t * segments;
  const int64_t base = all / ranges, extra = all % ranges;
  std::vector<int64_t> words(4 * (ranges + 1), 0);
  int64_t* const where = words.data();
  for (int64_t x = 0; x < ranges; ++x) {
    const int64_t t0 = range_start(x, 1, base, extra);
    RangeBegin r = t0 >= all ? no_row(t0) : find_begin(t0, 0, rows, 0, [&](int64_t i) { return tiles[i] * segments; });
    if (t0 < all) {   // the segment of the row
      const int64_t p = r.tiles / segments, segment = (t0 - r.first) / p;
      r = RangeBegin{r.place * segments + segment, r.first + segment * p, p, t0};
    }
    put_record(where, x, r);
  }
  where[4 * ranges + 3] = all;

  // what has to be joined: the segments that lie in several ranges, and those ranges
  std::map<int64_t, std::vector<int64_t>> want;
  int64_t line = 0;
  for (int64_t i = 0; i < rows; ++i)
    for (int64_t s = 0; s < segments; ++s, line += tiles[i]) {
      std::vector<int64_t> in;
      for (int64_t x = 0; x < ranges; ++x) {
        const int64_t t0 = begin_of(where, x), t1 = begin_of(where, x + 1);
        if (t0 < t1 && t0 < line + tiles[i] && t1 > line) in.push_back(x);
      }
      if (in.size() > 1) want[i * segments + s] = in;
    }

  auto parts = [&](int64_t x) {   // of the join on behalf of range x
    std::vector<int64_t> in;
    const int64_t end = record_of(where, x).first + record_of(where, x).tiles;
    for (int64_t i = 0; i <= ranges - x && begin_of(where, x - 1 + i) < end; ++i)
      if (begin_of(where, x + i) > begin_of(where, x - 1 + i)) in.push_back(x - 1 + i);
    return in;
  };
  int bad = 0;
  std::map<int64_t, std::vector<int64_t>> one, sixteen;
  for (int64_t x = 1; x < ranges; ++x)
    if (cuts_first(record_of(where, x), begin_of(where, x - 1))) {
      if (one.count(where[4 * x])) ++bad;
      one[where[4 * x]] = parts(x);
    }
  for (int64_t place = 0; place < rows * segments; ++place) {
    int64_t found = ranges;
    for (int64_t i = ranges - 1; i >= 1; --i)
      if (where[4 * i] == place && begins_inside(record_of(where, i))) found = i;
    if (found < ranges && cuts_first(record_of(where, found), begin_of(where, found - 1))) sixteen[place] = parts(found);
  }
  if (bad || one != want || sixteen != want) {
    std::printf("%s: %lld rows, %lld segments, %lld tiles, %lld ranges: %zu to join, %zu and %zu joined\n", what,
                (long long)rows, (long long)segments, (long long)all, (long long)ranges, want.size(), one.size(), sixteen.size());
    return 1;
  }
  return 0;
}

int main() {
  int bad = 0;
  // totals around nothing and the number of ranges, the tiles in one row of several
  for (int64_t ranges : {2, 3, 8, 147, 148})
    for (int64_t total : {int64_t(0), int64_t(1), int64_t(2), int64_t(3), ranges - 1, ranges, ranges + 1, 2 * ranges + 1})
      for (int64_t rows : {1, 2, 9, 16, 301})
        for (int64_t at : {int64_t(0), rows / 2, rows - 1})
          for (int64_t segments : {1, 3}) {
            std::vector<int64_t> t(rows, 0);
            t[at] = total;
            bad += batch(t, segments, ranges, "one row");
          }
  for (int n = 0; n < 20000; ++n) {
    const int64_t rows = 1 + draw(n % 2 ? 6 : 40), most = 1 + draw(n % 3 ? 3 : 30), empty = draw(4);
    std::vector<int64_t> t(rows);
    for (auto& x : t) x = draw(4) < empty ? 0 : draw(most + 1);
    bad += batch(t, 1 + draw(3), 2 + draw(60), "random");
    if (bad > 20) break;
  }
  std::printf("%d batches wrong\n", bad);
  return bad != 0;
}
"""


def test_joins_take_the_cut_rows_only(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    source = tmp_path / "ranges.cpp"
    source.write_text(PROGRAM)
    program = tmp_path / "ranges"
    built = subprocess.run([cxx, "-std=c++17", "-O1", "-x", "c++", "-I", str(CSRC), str(source), "-o", str(program)],
                           capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([str(program)], capture_output=True, text=True, timeout=120)
    assert ran.returncode == 0, ran.stdout
