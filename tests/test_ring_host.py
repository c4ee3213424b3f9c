"""The bookkeeping of a kernel that gives up (csrc/ring.cuh): which phase of which barrier its last
loads complete.  Compiled for the host; at every point where a producer may stop, the phases are
compared with a plain count of the loads per barrier."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "featgraph_b200", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "ring.cuh"
int main() {
  for (uint32_t slots = 1; slots <= 14; ++slots) {
    fg::Place place;
    uint32_t count[14] = {};
    for (uint32_t loaded = 0; loaded < 100; ++loaded) {
      for (uint32_t k = 0; k < (loaded < slots ? loaded : slots); ++k)
        if (fg::last_round(place, k) != ((count[k] - 1) & 1))
          return printf("slots %u loaded %u slot %u\n", slots, loaded, k), 1;
      if (place.at != loaded % slots || place.parity != (loaded / slots & 1))
        return printf("place of load %u of %u slots\n", loaded, slots), 1;
      ++count[place.at];
      place.next(slots);
    }
  }
  // a producer of items: the rows of an item are loaded once, before its steps.  It may stop before
  // the rows, or at any step behind them: the last rows that were issued are item `item` - 1's in
  // the first case and item `item`'s in the second.
  fg::Loads rows;
  if (rows.any()) return printf("nothing issued\n"), 1;
  for (uint32_t item = 0; item < 9; ++item) {
    if (item > 0 && (!rows.any() || rows.last_parity() != ((item - 1) & 1)))
      return printf("stopped before the rows of item %u\n", item), 1;
    ++rows.issued;
    if (!rows.any() || rows.last_parity() != (item & 1))
      return printf("stopped in the steps of item %u\n", item), 1;
  }
  return 0;
}
"""


def test_what_a_kernel_that_gives_up_waits_for(tmp_path):
    source = tmp_path / "ring.cpp"
    source.write_text(PROGRAM)
    binary = str(tmp_path / "ring")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(source), "-o", binary], check=True)
    done = subprocess.run([binary], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
