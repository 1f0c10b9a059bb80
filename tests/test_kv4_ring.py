"""The ring of copies of the 4-bit attention, run on the host: whichever wait gives up, every copy
that was issued is waited for, nothing is used or issued after that, and without one every stage is
used once, in order, after its own copy."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "proof-carrying-kernels_b200" / "csrc"

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "kv4_ring.h"

// One run: the wait number `fails` (-1: none) gives up. Counts what was issued, waited for and used.
template <int kSlots>
bool run(int stages, int fails) {
  std::vector<int> holds(kSlots, -1), waited(stages, 0), used(stages, 0);
  int issued = 0, waits = 0, next = 0;
  bool gone = false, ok = true;
  for (; issued < kSlots && issued < stages; ++issued) holds[issued] = issued;
  const bool alive = pck::take_stages<kSlots>(
      stages,
      [&](int slot) {
        ok = ok && holds[slot] >= 0;
        if (holds[slot] >= 0) ++waited[holds[slot]];
        if (gone || fails == waits) holds[slot] = -1;
        gone = gone || fails == waits;
        return waits++ != fails;
      },
      [&](int k, int slot) {
        ok = ok && !gone && holds[slot] == k && next == k;
        ++next;
        ++used[k];
      },
      [&](int k, int slot) {
        ok = ok && !gone && k == issued && holds[slot] == k - kSlots;
        holds[slot] = k;
        ++issued;
      });
  ok = ok && alive == (fails < 0 || fails >= waits);
  for (int k = 0; k < stages; ++k) ok = ok && waited[k] == (k < issued) && (!alive || used[k] == 1);
  return ok;
}

template <int kSlots>
bool all() {
  for (int stages = 0; stages <= 4 * kSlots + 3; ++stages) {
    for (int fails = -1; fails < stages; ++fails) {
      if (!run<kSlots>(stages, fails)) {
        std::printf("slots %d, stages %d, wait %d\n", kSlots, stages, fails);
        return false;
      }
    }
  }
  return true;
}

int main() { return all<1>() && all<2>() && all<5>() && all<12>() && all<16>() ? 0 : 1; }
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host compiler")
def test_every_copy_that_was_issued_is_waited_for(tmp_path: Path) -> None:
    source = tmp_path / "ring.cpp"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{CSRC}", str(source), "-o", str(tmp_path / "ring")], check=True)
    done = subprocess.run([str(tmp_path / "ring")], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout


def test_the_attention_takes_its_stages_through_the_ring() -> None:
    """The kernel has no wait on its copies beside the one that it hands to the ring."""
    text = (CSRC / "kv4_attention.cu").read_text()
    assert text.count("take_stages<") == 1 and text.count("mbar_wait(") == 1
