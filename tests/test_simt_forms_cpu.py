"""The any-shape attention's choice of a layout, compiled for the host: two CTAs of it share an SM at every shape where two
CTAs of unpadded tiles (Q, K, V of 64 rows, P of 64 x 65 and the bias rows) would."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")

PROGRAM = r"""
#include <stdio.h>
#include "common.cuh"
#include "relpos_simt.cuh"
int main() {
  using namespace samrs;
  int bad = 0, forms[3] = {0, 0, 0};
  for (int h = 1; h <= 128; ++h)
    for (int w = 1; w <= 128; ++w)
      for (int hd = 1; hd <= 128; ++hd) {
        const SimtForm form = simt_form(h, w, hd);
        const long sm = 228 * 1024, reserved = 1024, own = 4 * (long)simt_smem_floats(form, h, w, hd) + reserved;
        const long unpadded = 4 * (3L * 64 * hd + 64 * 65 + 64L * (h + w)) + reserved;
        ++forms[form];
        bad += 2 * unpadded <= sm && 2 * own > sm;
        bad += own > 227 * 1024 + reserved;                    // every shape runs
        bad += form == kSimtTiny && h * w > 64;                // one tile
      }
  printf("%d %d %d %d\n", bad, forms[0] > 0, forms[1] > 0, forms[2] > 0);
  return 0;
}
"""


def test_two_ctas_where_unpadded_tiles_would_fit_twice(tmp_path):
    if not os.path.exists(NVCC):
        pytest.skip("no nvcc")
    src, exe = tmp_path / "forms.cu", tmp_path / "forms"
    src.write_text(PROGRAM)
    subprocess.run([NVCC, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr",
                    "-I", os.path.join(ROOT, "sam-rs_b200", "csrc"), "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()
    assert out == ["0", "1", "1", "1"]
