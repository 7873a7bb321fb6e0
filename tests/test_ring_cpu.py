"""The ring of loads of moa_b200/csrc/ring.h with a model of its barriers, compiled for the CPU.

The model is a barrier that takes one arrival a phase, and loads that land after so many waits, or never.  It holds the
ring to what the hardware asks for: a stage is armed only when its barrier's phase is closed and its load has landed, a wait
is for the phase that is open, and when the warp is through every load was waited for, whether it came or not."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moa_b200", "csrc")
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include "ring.h"

// usage: UNITS LATE NEEDS: unit LATE's load lands at the NEEDS-th wait that looks for it (0: never), the others at the first
template <int kStages>
int run(int units, int late, int needs) {
  struct Bar { uint32_t phase = 0; bool open = false; int unit = -1, waits = 0; } bars[kStages];
  moa::Ring<kStages> ring;
  int asked = 0, taken = 0, ran_out = 0, waited = 0;
  bool more = units > 0;
  auto fail = [](const char* what) { std::puts(what); std::exit(1); };
  auto issue = [&](int stage) {
    if (more) {
      Bar& b = bars[stage];
      if (b.open) fail("armed while its phase is open");
      b.open = true;
      b.unit = asked++;
      b.waits = 0;
      more = asked < units;
    }
  };
  auto wait = [&](int stage, uint32_t parity) {
    Bar& b = bars[stage];
    ++waited;
    if (b.phase != parity) fail("waits for a phase that is over");
    if (!b.open) {                               // nothing is under way: the wait runs out
      if (!ring.late) fail("takes a load that nobody asked for");
      return false;
    }
    ++b.waits;
    if (b.unit == late && (needs == 0 || b.waits < needs)) {
      ++ran_out;
      return false;
    }
    b.phase ^= 1;
    b.open = false;
    return true;
  };
  for (int s = 0; s < kStages; ++s) issue(s);
  for (int u = 0; u < units; ++u) {            // the warp goes through all its units, late or not
    if (!ring.late) {
      const int stage = ring.stage;
      if (bars[stage].unit != u) fail("another unit's stage");
      ring.take(wait);
      if (ring.late) more = false;
      else ++taken;
    }
    issue(ring.stage);
    ring.next();
  }
  const bool was_late = ring.late;
  if (was_late) ring.drain(wait);
  for (const Bar& b : bars)
    if (b.open && (b.unit != late || b.waits < 2)) fail("a load is left without a wait");
  if (was_late != (late < units && needs != 1)) fail("late or not?");
  if (!was_late && (taken != units || waited != units)) fail("units");
  if (was_late && taken != late) fail("units before the late one");
  if (was_late && waited != late + 1 + kStages) fail("waits");
  return 0;
}

int main(int argc, char** argv) {
  const int most = std::atoi(argv[1]);
  for (int units = 0; units <= most; ++units)
    for (int late = 0; late <= units; ++late)
      for (int needs = 0; needs < 4; ++needs)
        if (run<2>(units, late, needs) || run<4>(units, late, needs) || run<1>(units, late, needs)) return 1;
  std::puts("ok");
}
"""


def _run(folder, header_folder):
    source, program = folder / "ring.cpp", folder / "ring"
    source.write_text(PROGRAM)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-Wno-unknown-pragmas", "-I", str(header_folder),
                    str(source), "-o", str(program)], check=True)
    return subprocess.run([str(program), "40"], text=True, capture_output=True, timeout=120)


def test_ring_arms_takes_and_drains(tmp_path):
    done = _run(tmp_path, CSRC)
    assert done.returncode == 0 and done.stdout == "ok\n", done.stdout


@pytest.mark.parametrize("right,wrong,what", [
    ("late = !wait(stage, parity);", "wait(stage, parity);", "armed while|without a wait"),     # on as if nothing had happened
    ("if (!late) advance();", "advance();", "phase that is over|without a wait"),
    ("for (int s = 0; s < kStages; ++s) {", "for (int s = 1; s < kStages; ++s) {", "without a wait|waits"),
    ("parity ^= 1;", "", "phase that is over"),
])
def test_the_model_sees_mistakes(tmp_path, right, wrong, what):
    text = open(os.path.join(CSRC, "ring.h")).read()
    assert text.count(right) == 1
    (tmp_path / "ring.h").write_text(text.replace(right, wrong))
    done = _run(tmp_path, tmp_path)
    assert done.returncode == 1 and re.search(what, done.stdout), done.stdout
