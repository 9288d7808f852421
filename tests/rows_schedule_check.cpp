// rows_schedule_check.cpp -- CPU replay of the loads, waits and reads of rows_tile.h's loop
// (welder_typical_chain_amd/csrc/rows_schedule.h), for every instance: a fragment is read only
// of a stage whose loads every wave had waited for at a barrier, and a stage is loaded only
// where every wave had left it at one.
//
// Build: g++ -std=c++17 -I<csrc> rows_schedule_check.cpp; prints "OK" and exits 0.  With -DLATE
// the replay is of an order whose last loads come behind the wait, which it must refuse.
#include <cstdio>
#include <deque>

#include "rows_schedule.h"

using namespace wtc::rows;

static int g_fail = 0;

// A stage's content in parts of one tensor's half: what a slot of the ring holds is
// `stage`, whole for this wave once it waited, for all waves behind the next barrier.
struct Part {
  int stage = -100;
  bool waited = false, common = false;
};

template <int ND, bool PREFIX, int A> struct Replay {
  using O = RowsSchedule<ND, PREFIX, A>;
#ifdef LATE
  static constexpr int AHEAD = O::STEPS;  // the barrier at step 0, before the step's loads
#else
  static constexpr int AHEAD = O::AHEAD;
#endif
  static constexpr int BARRIER = O::STEPS - AHEAD;
  Part ring[O::STAGES][2][O::TENSORS];  // slot, half, tensor (of the waves that load it)
  int left[O::STAGES];                  // the stage that every wave has left in a slot
  std::deque<Part*> flight;             // in their order
  int turn = 0;

  void fail(const char* what, int stage, int half, int y) {
    if (g_fail++ < 20) std::printf("ND %d PREFIX %d A %d turn %d: %s stage %d half %d step %d\n", ND, PREFIX, A, turn, what, stage, half, y);
  }
  int slot(int stage) const { return (stage + 1) % O::STAGES; }  // stages count from -1
  void load(int stage, int half, int tensor, int y) {
    Part& p = ring[slot(stage)][half][tensor];
    if (p.stage != -100 && left[slot(stage)] != p.stage) fail("loaded over", p.stage, half, y);
    p = Part{stage, false, false};
    flight.push_back(&p);
  }
  void wait() {  // the newest LOADING stages' loads stay in flight
    while ((int)flight.size() > O::LOADING * 2 * O::TENSORS) flight.front()->waited = true, flight.pop_front();
  }
  void barrier() {
    for (auto& s : ring)
      for (auto& h : s)
        for (Part& p : h) p.common |= p.waited;
  }
  void read(int stage, int half, int y) {  // keys and values go alike; of one tensor a wave, both waves do
    const int tensor = O::TENSORS == 2 ? y / O::FRAGS : 0;
    const Part& p = ring[slot(stage)][half][tensor];
    if (p.stage != stage || !p.common) fail("read before it landed", stage, half, y);
    if (left[slot(stage)] == stage) fail("read after it was left", stage, half, y);
  }
  void run() {
    for (int& x : left) x = -100;
    for (int x = 0; x < O::STAGES; ++x) {
      if (x == O::STAGES - 1) wait(), barrier();
      for (int t = 0; t < O::TENSORS; ++t)
        for (int h = 0; h < 2; ++h) load(x - 1, h, t, -1);
    }
    for (int y = 0; y < O::FRAGS; ++y) read(-1, 1, y);  // unit 0's scores
    wait(), barrier();
    left[slot(-1)] = -1;
    int stage = 0;
    for (int y = 0; y < AHEAD; ++y) read(stage, 0, y);
    for (turn = 0; turn < 12; ++turn)
      for (int x = 0; x < 2; ++x)
        for (int y = 0; y < O::STEPS; ++y) {
          if (x == 1 && y == BARRIER) wait(), barrier(), left[slot(stage)] = stage, ++stage;
          if (y + AHEAD < O::STEPS) read(stage, x, y + AHEAD);
          else read(stage, x ^ 1, y + AHEAD - O::STEPS);
          if (PREFIX) {
            if (y == O::FIRST) load(turn + O::STAGES - 1, x, 0, y);
            if (y == O::SECOND && O::TENSORS == 2) load(turn + O::STAGES - 1, x, 1, y);
          } else if (x < O::TENSORS && y == (x ? O::SECOND : O::FIRST)) {
            for (int h = 0; h < 2; ++h) load(turn + O::STAGES - 1, h, x, y);
          }
        }
  }
};

template <int ND> void all() {
  Replay<ND, true, 1>().run();
  Replay<ND, true, 2>().run();
  Replay<ND, false, 1>().run();
  Replay<ND, false, 2>().run();
}

int main() {
  all<1>();
  all<2>();
  all<3>();
  all<4>();
  if (g_fail) return std::printf("%d failures\n", g_fail), 1;
  std::printf("OK\n");
  return 0;
}
