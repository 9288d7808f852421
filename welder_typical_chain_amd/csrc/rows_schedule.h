// rows_schedule.h -- the order of loads, waits and reads in rows_tile.h's loop, as numbers
// that a host program can replay.
//
// A turn of the loop has two halves x of STEPS steps y; a step uses one fragment of a stage,
// read AHEAD steps before (so a half's last AHEAD steps read the next half's first fragments).
// At step BARRIER of half 1 all of the turn's stage is read: the wave waits until of its
// loads only those of the newest LOADING stages may be in flight and meets the others, which
// makes the next stage whole.  The count holds only if this turn's own loads, of the stage
// after the next one, are all issued before it.
#pragma once

namespace wtc {
namespace rows {

// ND: 32-column subtiles of dim; A: row blocks of 32 a wave, which loads keys and values (2)
// or one of them (1).
template <int ND, bool PREFIX, int A> struct RowsSchedule {
  static constexpr int STAGES = 3, LOADING = STAGES - 2;
  static constexpr int TENSORS = A == 2 ? 2 : 1;
  static constexpr int FRAGS = 2 * ND, STEPS = 2 * FRAGS;  // of a half: fragments of keys, then as many of values
  // (of 4 steps, 4 ahead would leave none for the loads of half 1)
  static constexpr int AHEAD = A == 1 && !(PREFIX && ND == 1) ? 4 : 3;
  static constexpr int BARRIER = STEPS - AHEAD;
  // Steps that load a wave's first and second tensor.  PREFIX: half x of the stage at half x;
  // otherwise all of the first tensor at half 0, of the second at half 1.
  static constexpr int FIRST = PREFIX && BARRIER > 2 ? 1 : 0, SECOND = PREFIX && BARRIER > 2 ? 2 : 0;
  static constexpr int LAST = TENSORS == 2 ? SECOND : PREFIX ? FIRST : -1;  // of half 1 that loads
  static_assert(LAST < BARRIER, "a stage's loads are issued before the wait that counts them");
  static_assert(BARRIER >= 0, "a fragment is read at most one half ahead");
};

}  // namespace rows
}  // namespace wtc
