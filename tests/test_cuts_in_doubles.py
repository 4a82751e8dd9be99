"""Cuts of a line formed in doubles (csrc/sp_paged_plan.h): the device has no division there but a reciprocal to 2^-24 and one step that squares its error.  The same
arithmetic on the CPU, from reciprocals that are off by as much as that in either direction: the cuts are the quotients all the same."""

import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "shareprefill_amd", "csrc")
PROGRAM = """
#include <math.h>
#include <stdio.h>
#include "sp_paged_plan.h"
int main() {
  uint64_t x = 1;
  long bad = 0;
  const double offs[] = {0.0, 0x1p-24, -0x1p-24, 0x1p-25, -0x1p-25, 0x1.8p-26, -0x1.4p-28};
  for (int i = 0; i < 20000; ++i) {
    x = x * 6364136223846793005ull + 1442695040888963407ull;
    const int parts = 1 + (int)(x >> 40) % 512;
    // lengths below 2^36: any, multiples of the parts, and one to either side of those, where a quotient is nearest to a whole number
    int64_t total = (int64_t)((x >> 8) & ((1ull << (1 + i % 36)) - 1));
    if (i % 4) total = total / parts * parts + i % 4 - 2;
    if (total < 0) total = 0;
    PgCuts cuts = pg_cuts(total, parts);
    for (double off : offs) {
      const double r = 1.0 / parts * (1.0 + off);
      cuts.inverse = fma(fma(-(double)parts, r, 1.0), r, r);
      for (int p = 0; p <= parts + 1; ++p) bad += pg_cut_at(cuts, p) != (p > parts ? total : (int64_t)((unsigned __int128)total * p / parts));
    }
  }
  printf("%ld\\n", bad);
}
"""


def test_reciprocals_that_are_off(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    (tmp_path / "cuts.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-Wall", "-ffp-contract=off", "-I", CSRC, str(tmp_path / "cuts.cpp"), "-o", str(tmp_path / "cuts")], check=True)
    assert subprocess.run([str(tmp_path / "cuts")], capture_output=True, text=True, check=True).stdout.strip() == "0"
