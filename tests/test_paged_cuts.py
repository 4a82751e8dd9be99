"""The cuts of a line of row tiles, or of single tokens' sequences, with the units that the kernels count (csrc/sp_paged_plan.h), on the CPU: every
block is some workgroup's, and the notes that workgroups leave lead the merging launch to all parts of what was cut and to no others."""

import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "shareprefill_amd", "csrc")
PROGRAM = """
#include <stdio.h>
#include <vector>
#include "sp_paged_plan.h"
int main() {
  int which, n, room;
  while (scanf("%d %d %d", &which, &n, &room) == 3) {
    const int overhead = which ? PD_OVERHEAD : PG_OVERHEAD, share = which ? PD_MIN_SHARE : PG_MIN_SHARE;
    std::vector<int> blocks(n);
    int64_t total = 0;
    for (int& b : blocks) {
      scanf("%d", &b);
      total += b + overhead;
    }
    const int64_t parts = pg_parts(total, room, share);
    printf("%d %d %ld", overhead, pg_near(total, parts), (long)parts);
    for (int64_t p = 0; p <= parts; ++p) {
      const int64_t cut = p < parts ? pg_cut(total, parts, p) : total;
      int x = 0;
      int64_t at = 0;
      while (x < n && cut >= at + blocks[x] + overhead) at += blocks[x++] + overhead;
      int tile = 0;
      if (x < n) {
        tile = pg_snap(cut - at, blocks[x], overhead, pg_near(total, parts));
        if (tile >= blocks[x] && tile != 0) ++x, tile = 0;
      }
      printf(" %d %d", x, tile);
    }
    printf("\\n");
  }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    tmp = tmp_path_factory.mktemp("cuts")
    (tmp / "cuts.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-Wall", "-Werror", "-Wno-unused-function", "-Wno-unused-result", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", CSRC, str(tmp / "cuts.cpp"), "-o", str(tmp / "cuts")], check=True)

    def run(lines):
        text = "".join("%d %d %d\n%s\n" % (which, len(blocks), room, " ".join(map(str, blocks))) for which, blocks, room in lines)
        out = subprocess.run([str(tmp / "cuts")], input=text, capture_output=True, text=True, check=True).stdout
        return [list(map(int, line.split())) for line in out.splitlines()]

    return run


@pytest.mark.parametrize("which", [0, 1], ids=["row tiles", "single tokens"])
def test_notes_lead_to_every_part(ask, which):
    rng = random.Random(which)
    lines = [(which, [0], 8), (which, [1], 8), (which, [0, 0, 0], 64), (which, [100000], 256), (which, [1] * 500, 256), (which, [3, 4, 5] * 60, 32)]
    for _ in range(400):
        blocks = [rng.choice((0, 1, 2, 3, rng.randrange(1, 12), rng.randrange(1, 300))) for _ in range(rng.randrange(1, 60))]
        lines.append((which, blocks, rng.choice((1, 2, 5, 32, 64, 256))))
    cut_tiles = 0
    for (_, blocks, room), (overhead, near, parts, *flat) in zip(lines, ask(lines)):
        places = list(zip(flat[::2], flat[1::2]))
        assert 1 <= parts <= room and len(places) == parts + 1
        assert places[0] == (0, 0) and places[-1] == (len(blocks), 0) and places == sorted(places)
        covered = [[] for _ in blocks]  # (workgroup, first, last) of every row tile, in order
        notes = []
        for w, ((x0, t0), (x1, t1)) in enumerate(zip(places, places[1:])):
            note = ["none", None]  # what its first row tile's part is, the row tile that starts here and goes on
            for x in range(x0, x1 + (t1 > 0)):
                first, last = (t0 if x == x0 else 0), (t1 if x == x1 else blocks[x])
                covered[x].append((w, first, last))
                if (first, last) != (0, blocks[x]):
                    if first == 0:
                        note[1] = x
                    else:
                        note[0] = "last" if last == blocks[x] else "middle"
            notes.append(note)
        for x, n in enumerate(blocks):
            assert covered[x][0][1] == 0 and covered[x][-1][2] == n
            assert all(a[2] == b[1] and a[0] + 1 == b[0] for a, b in zip(covered[x], covered[x][1:]))
            assert all(a < b for _, a, b in covered[x]) or n == 0
            if len(covered[x]) > 1:
                cut_tiles += 1
                w0 = covered[x][0][0]
                assert notes[w0][1] == x
                count = 1  # what the merging launch finds
                while True:
                    count += 1
                    if notes[w0 + count - 1][0] != "middle":
                        break
                assert count == len(covered[x]) and notes[w0 + count - 1][0] == "last"
                assert all(near <= t <= n - near for _, _, t in covered[x][:-1])
    assert cut_tiles > 1000
