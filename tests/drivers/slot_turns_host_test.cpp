// Runs the order in which the linear layers' epilogue takes and leaves its slot of
// shared memory (7_b200/csrc/slot_turns.h) against bulk groups that complete as late
// as they may: whoever takes a place must find no store that still reads it.
// Plain g++, no CUDA.  Prints the places taken too early; exits 1 if there are any.
#include "slot_turns.h"

#include <cstdio>
#include <random>
#include <vector>

namespace {

// A thread's bulk groups, oldest first: each holds the places its stores read.
struct Late {
  struct State {
    std::vector<std::vector<const uint8_t *>> pending;
    std::vector<const uint8_t *> open; // stores not yet in a group
  };
  State *s;
  template <int N> void wait_read() const { // all but the newest N groups have read their source
    while (s->pending.size() > N)
      s->pending.erase(s->pending.begin());
  }
  void commit() const {
    s->pending.push_back(s->open); // (empty where nothing was stored)
    s->open.clear();
  }
  bool reads(const uint8_t *place) const {
    for (const auto &g : s->pending)
      for (const uint8_t *p : g)
        if (p == place)
          return true;
    for (const uint8_t *p : s->open)
      if (p == place)
        return true;
    return false;
  }
};

// `stored(i)`: whether use i leaves by a bulk store.
template <bool kHalves, typename F> int early(int uses, F stored) {
  static uint8_t memory[2];
  uint8_t *slot = memory;
  int other = 1, bad = 0;
  Late::State state;
  const Late bulk{&state};
  for (int i = 0; i < uses; ++i) {
    wave::linear_detail::slot_take<kHalves>(slot, other, bulk);
    bad += bulk.reads(slot); // it is written from here on
    if (stored(i))
      state.open.push_back(slot);
    wave::linear_detail::slot_leave(bulk);
  }
  return bad;
}

} // namespace

int main() {
  int total = 0;
  auto say = [&](const char *what, int bad) {
    std::printf("%s: %d\n", what, bad);
    total += bad;
  };
  say("all stored", early<true>(100, [](int) { return true; }));
  say("z stored, y direct", early<true>(100, [](int i) { return i % 2 == 0; }));
  say("z direct, y stored", early<true>(100, [](int i) { return i % 2 == 1; }));
  say("whole blocks, then a cut one", early<true>(100, [](int i) { return i % 10 < 8; }));
  say("a narrow last chunk", early<true>(100, [](int i) { return i % 6 < 4; }));
  say("one whole use", early<true>(100, [](int i) { return i % 7 == 0; }));
  std::mt19937 rng(1);
  for (int rep = 0; rep < 1000; ++rep) {
    const unsigned one_in = 2 + rep % 9;
    total += early<true>(200, [&](int) { return rng() % one_in != 0; });
    total += early<false>(200, [&](int) { return rng() % one_in != 0; });
  }
  std::printf("taken too early: %d\n", total);
  return total != 0;
}
