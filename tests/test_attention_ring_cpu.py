"""CPU: the attention kernels' rings of buffers when a wait gives up (csrc/ring.cuh).

A program built from the header walks pages as a warp of the 8-bit attention does --
keys, values and the next page's keys in three buffers, some pages outside the cache --
over barriers that count boxes, with every wait in turn giving up while its box is still
under way, and later ones giving up too or not.  The warp ends its page, or leaves it at
once.  No box may be sent to a buffer that waits for one, every wait has to be for the
phase of the box under way, and all boxes have to have landed at the end."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "10_20_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <vector>

#include "ring.cuh"

using v1x::attn::RingState;

static int bad = 0;

struct Barriers {
  int landed[3] = {0, 0, 0};
  bool flying[3] = {false, false, false};
  int waits = 0, give_up_at;
  bool later;
  Barriers(int at, bool later) : give_up_at(at), later(later) {}
  void send(int slot) {
    if (flying[slot]) ++bad;      // two boxes in one phase
    flying[slot] = true;
  }
  bool wait(int slot, unsigned parity, bool drain) {
    if (!flying[slot] || parity != (landed[slot] & 1u)) {
      ++bad;                      // a wait that no box ends, or for another phase
      return true;
    }
    if (!drain) {
      const int n = waits++;
      if (n == give_up_at || (later && n > give_up_at)) return false;
    }
    flying[slot] = false;
    ++landed[slot];
    return true;
  }
};

// here[i]: page i is in the cache
static int walk(const std::vector<bool>& here, int give_up_at, bool leave, bool later) {
  Barriers b(give_up_at, later);
  RingState ring;
  const int n = here.size();
  auto load = [&](int slot, int page) {
    if (page >= n || !here[page] || !ring.start(slot)) return;
    b.send(slot);
  };
  auto arrived = [&](int slot) {
    const bool done = b.wait(slot, ring.phase(slot), false);
    ring.waited(slot, done);
    return done;
  };
  load(0, 0);
  load(1, 0);
  load(2, 1);
  for (int it = 0, slot = 0; it < n && ring.ok; ++it) {
    const int vslot = (slot + 1) % 3;
    if (here[it]) {
      if (!arrived(slot) && leave) break;
      load(slot, it + 1);
      if (!arrived(vslot) && leave) break;
    } else {
      load(slot, it + 1);
    }
    load(vslot, it + 2);
    slot = (vslot + 1) % 3;
  }
  if (!ring.ok)
    for (int i = 0; i < 3; ++i)
      if (ring.under_way(i)) b.wait(i, ring.phase(i), true);
  for (int i = 0; i < 3; ++i)
    if (b.flying[i]) ++bad;       // lands after its CTA
  return b.waits;
}

int main() {
  for (int n = 1; n <= 9; ++n)
    for (int mask = 0; mask < 1 << n; ++mask) {
      std::vector<bool> here(n);
      for (int i = 0; i < n; ++i) here[i] = mask >> i & 1;
      const int waits = walk(here, 1 << 20, true, true);
      for (int at = 0; at < waits; ++at)
        for (bool leave : {true, false})
          for (bool later : {true, false}) walk(here, at, leave, later);
    }
  std::printf("%d faults\n", bad);
  return bad != 0;
}
"""


# The prompt attention's producer: whole tiles by boxes, a last partial one by copies, into
# buffers in turn; the consumers free them in order, up to a place where they give up.
PROMPT = r"""
#include <cstdio>

#include "ring.cuh"

int main() {
  constexpr int kSlots = 3;
  int bad = 0;
  for (int whole = 0; whole <= 14; ++whole)
    for (int rest = 0; rest <= 2; rest += 2)            // keys and values of the partial tile
      for (int freed = 0; freed <= whole + rest; ++freed)       // loads whose buffers become free
        for (int landed = freed; landed <= whole + rest; ++landed) {   // loads that have landed at the end
          v1x::attn::LastBoxes<kSlots> last;
          int phases[kSlots] = {0, 0, 0}, sent = 0;     // phases: loads of a buffer that have landed
          int box_in[kSlots] = {-1, -1, -1};            // the load whose box a buffer got last
          for (int u = 0; u < whole + rest; ++u) {
            const int slot = u % kSlots, turn = u / kSlots;
            if (u >= kSlots && u - kSlots >= freed) break;      // the wait for the buffer gives up
            if (u < whole) {
              last.box(slot, turn);
              box_in[slot] = u;
            } else {
              last.copy(slot);
              box_in[slot] = -1;
            }
            ++sent;
          }
          for (int u = 0; u < sent && u < landed; ++u) ++phases[u % kSlots];
          for (int i = 0; i < kSlots; ++i) {
            const int turn = last.turns[i];
            // a box under way is waited for, in its own phase; a wait's phase is the current or the last one
            if (box_in[i] >= landed && turn != box_in[i] / kSlots) ++bad;
            if (turn >= 0 && phases[i] != turn && phases[i] != turn + 1) ++bad;
          }
        }
  std::printf("%d faults\n", bad);
  return bad != 0;
}
"""


@pytest.mark.parametrize("program", [PROGRAM, PROMPT], ids=["decode", "prompt"])
def test_a_wait_that_gives_up_leaves_no_box_behind(tmp_path, program):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host compiler")
    source = tmp_path / "ring.cpp"
    source.write_text(program)
    binary = tmp_path / "ring"
    built = subprocess.run([cxx, "-std=c++17", "-O1", "-x", "c++", "-I", str(CSRC), str(source), "-o", str(binary)],
                           capture_output=True, text=True)
    assert built.returncode == 0, built.stderr
    ran = subprocess.run([str(binary)], capture_output=True, text=True, timeout=120)
    assert ran.returncode == 0, ran.stdout
