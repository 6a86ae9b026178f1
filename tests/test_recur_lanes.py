"""Which words of other tiles the recurrence's lanes wait for, and what they read of a row, on the CPU: the kernels'
own function, compiled for the host."""

from __future__ import annotations

import pathlib
import subprocess

from plastax_amd import build

PROGRAM = """
#include "px_recur.h"
#include <cstdio>

template <int FORM>
int check(int units) {
  for (unsigned first = 0; first < static_cast<unsigned>(units); first += px::kSlab) {
    const unsigned end = first + px::kSlab < static_cast<unsigned>(units) ? first + px::kSlab : units;
    unsigned next = first;  // the units of the slab are the lanes' in order, each once
    for (int lane = 0; lane < 64; ++lane) {
      const px::Lane l = px::lane_of<FORM>(first, lane, units);
      bool fine = l.word >= first && l.word < end && l.next >= first && l.next < end;
      if (l.n > 0) fine &= l.col == next++ && l.word == l.col;
      if (l.n > 1) fine &= l.next == next++;
      if (FORM != px::kOne) fine &= l.at + 2 <= static_cast<unsigned>(units);
      if (FORM != px::kOne && l.n > 0) fine &= l.at == (l.n == 1 ? l.col - 1 : l.col);
      if (!fine) {
        std::printf("units %d, slab %u, lane %d: waits for %u and %u, reads %u\\n", units, first, lane, l.word, l.next, l.at);
        return 1;
      }
    }
    if (next != end) return std::printf("units %d, slab %u: %u units\\n", units, first, next - first), 1;
  }
  return 0;
}

int main() {
  if (check<px::kOne>(1)) return 1;
  for (int units = 2; units <= 700; ++units)
    if (units % 2 ? check<px::kOdd>(units) : check<px::kEven>(units)) return 1;
  for (int units : {1003, 4096, 4097, 8388607, 8388608})
    if (units % 2 ? check<px::kOdd>(units) : check<px::kEven>(units)) return 1;
  return 0;
}
"""


def test_tiles_wait_for_words_of_their_own_slab(tmp_path: pathlib.Path) -> None:
    """Tiles are taken in order slab by slab. A lane without a unit (past an odd or a last slab's end) that waited for
    another slab's word would wait for a tile that nothing says has been taken."""
    source, program = tmp_path / "lanes.hip", tmp_path / "lanes"
    source.write_text(PROGRAM)
    subprocess.run([build.hipcc(), "-x", "hip", "--offload-host-only", "-std=c++17", "-O1", "-I", str(build.CSRC),
                    str(source), "-o", str(program)], check=True, capture_output=True, text=True)
    ran = subprocess.run([str(program)], capture_output=True, text=True)
    assert ran.returncode == 0, ran.stdout
