// The ring of page copies of the single-token attention kernel
// (bitnetrs_b200/csrc/kvq_ring.h), driven as the kernel drives it, with the wait
// for a stage running out at every possible place: what is left in flight is
// waited for, stage by stage, each with the parity of its own copy.
#include <cstdio>
#include <vector>

#include "../bitnetrs_b200/csrc/kvq_ring.h"

static long checks = 0, faults = 0;
static void check(bool ok) {
  ++checks;
  faults += !ok;
}

// Units of `pairs` page pairs one after the other; the wait for pair `fails` (counted over all units) runs out.
template <int STAGES>
static void run(const std::vector<int>& units, int fails) {
  bitnet::StageRing<STAGES> ring;
  int copies[STAGES] = {}, landed[STAGES] = {};  // a stage's copies so far, and those waited for
  int seen = 0;
  auto fetch = [&](int i, int pairs) {
    if (i >= pairs) return;
    check(copies[ring.fill] == landed[ring.fill]);  // what was there has been used
    ++copies[ring.fill];
    ring.fetched();
  };
  auto wait = [&] {  // the phase that is waited for is that of the stage's one copy in flight
    check(copies[ring.take] == landed[ring.take] + 1 && ring.parity == (uint32_t)(landed[ring.take] & 1));
    ++landed[ring.take];
  };
  bool failed = false;
  for (int pairs : units) {
    for (int i = 0; i < STAGES; ++i) fetch(i, pairs);
    for (int i = 0; i < pairs && !failed; ++i) {
      if (seen++ == fails) {
        failed = true;
        break;
      }
      wait();
      ring.used();
      fetch(i + STAGES, pairs);
    }
    if (failed) {
      while (ring.flying) {
        wait();
        ring.used();
      }
      break;
    }
    check(ring.flying == 0);
  }
  for (int i = 0; i < STAGES; ++i) check(copies[i] == landed[i]);  // nothing is in flight at the end
}

template <int STAGES>
static void all() {
  for (int a = 1; a <= 3 * STAGES; ++a)
    for (int b = 0; b <= 2 * STAGES + 1; ++b)
      for (int fails = 0; fails <= a + b; ++fails) run<STAGES>({a, b, 1}, fails);
}

int main() {
  all<1>();
  all<2>();
  all<3>();
  all<4>();
  std::printf("checks %ld faults %ld\n", checks, faults);
  return faults != 0;
}
