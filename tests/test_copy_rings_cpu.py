"""What a producer waits for before its CTA may leave, on the CPU: the copies that it has armed and that nobody has been seen
to wait for, and no phase that it never armed."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "sam-rs_b200", "csrc")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

# The walk of the attention's dQ producer: rows of a tile on one barrier, steps on a ring, either given up at any wait. A
# barrier's current phase is the number of its arms so far; parity p names its last phase if (arms - 1) & 1 == p.
PROGRAM = r"""
#include <stdio.h>
#include "common.cuh"
#include "sm100.cuh"
using samrs::sm100::Armed;
int main() {
  int bad = 0, runs = 0;
  for (int stages = 1; stages <= 6; ++stages)
    for (int tiles = 1; tiles <= 4; ++tiles)
      for (int steps = 1; steps <= 9; ++steps)
        for (int quit = 0; quit <= tiles * (steps + 1); ++quit, ++runs) {
          Armed rows, ring;
          int row_arms = 0, arms[6] = {0}, left = quit, st = 0;
          bool okk = true;
          for (int tl = 0; tl < tiles && okk; ++tl) {
            if (left-- == 0) break;
            ++row_arms, ++rows.n;
            for (int s = 0; s < steps; ++s, ++ring.n) {
              if (left-- == 0) { okk = false; break; }
              ++arms[st];
              st = (st + 1) % stages;
            }
          }
          int seen_rows = 0, seen[6] = {0};
          rows.pending(1, [&](int k, unsigned parity) {
            bad += k != 0 || row_arms == 0 || parity != (unsigned)((row_arms - 1) & 1);
            ++seen_rows;
          });
          ring.pending(stages, [&](int k, unsigned parity) {
            bad += k < 0 || k >= stages || arms[k] == 0 || parity != (unsigned)((arms[k] - 1) & 1);
            ++seen[k];
          });
          bad += seen_rows != (row_arms > 0);
          for (int k = 0; k < stages; ++k) bad += seen[k] != (arms[k] > 0);
        }
  printf("%d %d\n", bad, runs > 1000);
  return 0;
}
"""


def test_armed_phases_are_the_ones_waited_for(tmp_path):
    if not os.path.exists(NVCC):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "rings.cu", tmp_path / "rings"
    src.write_text(PROGRAM)
    subprocess.run([NVCC, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr", "-I", CSRC,
                    "-o", str(exe), str(src)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split() == ["0", "1"]
