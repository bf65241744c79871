"""The waits for a ring's copies in flight, against a model of the ring: barriers that hold the phases of mbarriers, copies
that land late, a producer that stops at any point."""

import shutil
import subprocess
from pathlib import Path

import pytest

SOURCE = r"""
#include <cstdio>
#include <vector>
#include "copies.h"

struct Barrier {
  int phase = 0;        // phases completed
  int flying = 0;       // copies that complete the current one
  // a wait for a parity passes once the phase of that parity is over: the current one has the other parity
  bool passes(unsigned parity) const { return (static_cast<unsigned>(phase) & 1u) != parity; }
  void land() { if (flying) { flying = 0; ++phase; } }
};

int main() {
  for (int stages = 1; stages <= 5; ++stages)
    for (int issued = 0; issued <= 4 * stages + 3; ++issued)
      for (int late = 0; late <= stages; ++late) {  // this many of the last copies have not landed
        std::vector<Barrier> ring(stages);
        for (int i = 0; i < issued; ++i) {
          ring[i % stages].land();  // a stage is filled again after its last copy was consumed
          ring[i % stages].flying = 1;
        }
        for (int i = 0; i < issued - late; ++i)
          if (i >= issued - stages) ring[i % stages].land();
        int waits = 0;
        jc::for_last_copies(issued, stages, [&](int s, unsigned parity) {
          ++waits;
          // a wait that passes with the stage's copy in flight does not wait for it
          if (ring[s].flying && ring[s].passes(parity)) { std::printf("passes early: %d of %d\n", issued, stages); }
          ring[s].land();
          // one that does not pass once it has landed runs to its limit
          if (!ring[s].passes(parity)) { std::printf("never passes: %d of %d\n", issued, stages); }
        });
        for (auto& b : ring)
          if (b.flying) std::printf("left in flight: %d of %d\n", issued, stages);
        if (waits != (issued < stages ? issued : stages)) std::printf("%d waits: %d of %d\n", waits, issued, stages);
      }
  std::printf("done\n");
}
"""


def test_every_copy_in_flight_is_waited_for(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no C++ compiler")
    src, exe = tmp_path / "ring.cpp", tmp_path / "ring"
    src.write_text(SOURCE)
    csrc = Path(__file__).resolve().parent.parent / "jitcast_b200" / "csrc"
    subprocess.run(["g++", "-std=c++17", "-I", str(csrc), str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout == "done\n"
