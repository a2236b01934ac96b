// The bookkeeping of a ring of buffers that boxes land in, each behind a barrier of
// one phase a box.  Host and device; a warp's lanes hold it alike.
#pragma once

#include <stdint.h>

#include "ranges.cuh"

namespace v1x {
namespace attn {

struct RingState {
  uint32_t phases = 0;   // per buffer: the parity of the phase that the next wait is for
  uint32_t issued = 0;   // per buffer: a box is under way
  bool ok = true;        // no wait has given up

  // Whether a box may be sent to the buffer: it is under way from here on.  After a wait
  // that gave up none is, since the buffer's phase may not be complete.
  V1X_HD bool start(int slot) {
    if (!ok) return false;
    issued |= 1u << slot;
    return true;
  }
  V1X_HD uint32_t phase(int slot) const { return (phases >> slot) & 1; }
  V1X_HD bool under_way(int slot) const { return (issued >> slot) & 1; }
  // The wait for the buffer's box ended.  One that gave up changes nothing but `ok`: its
  // box may still land, in its phase, and has to be waited for before the CTA ends.
  V1X_HD void waited(int slot, bool done) {
    if (!done) {
      ok = false;
      return;
    }
    phases ^= 1u << slot;
    issued &= ~(1u << slot);
  }
};

// The box that each of a ring's buffers got last, where boxes and plain copies take turns
// in it: what may still be under way once all have been sent.
template <int kSlots>
struct LastBoxes {
  int turns[kSlots];     // the buffer's turn, whose phase the box ends; -1: no box since the last copy

  V1X_HD LastBoxes() {
    for (int& t : turns) t = -1;
  }
  V1X_HD void box(int slot, int turn) { set(slot, turn); }
  // A copy: its buffer was free, so the box before it has landed.
  V1X_HD void copy(int slot) { set(slot, -1); }

  V1X_HD void set(int slot, int turn) {
#ifdef __CUDA_ARCH__
#pragma unroll
#endif
    for (int i = 0; i < kSlots; ++i)
      if (i == slot) turns[i] = turn;
  }
};

}  // namespace attn
}  // namespace v1x
