"""How attention with shared starts of prompts is cut into work (csrc/sp_shared_plan.h, arithmetic that host and device share), on the CPU: the parts of a
line hold every step of every tile exactly once, a tile's parts lie side by side, and so do those of a request that waves go through step by step."""

import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "shareprefill_amd", "csrc")
PROGRAM = """
#include <stdio.h>
#include <vector>
#include "sp_shared_plan.h"
// items of `rows` rows and n steps a tile, the first `groups` of them groups, those from `streams` on waves'; room: workgroups.  Prints every piece: part (of a wave), item, tile, begin, end.
int main() {
  long items, groups, streams, room;
  while (scanf("%ld %ld %ld %ld", &items, &groups, &streams, &room) == 4) {
    std::vector<long> n(items), rows(items);
    std::vector<int64_t> line(items + 1);
    for (long i = 0; i < items; ++i) {
      if (scanf("%ld %ld", &n[i], &rows[i]) != 2) return 1;
      line[i + 1] = line[i] + (n[i] > 0 && rows[i] > 0 ? sh_units((int)n[i], (int)rows[i], i < groups ? SH_GROUP : i < streams ? SH_OWN : SH_STREAM) : 0);
    }
    const int64_t total = line[items], parts = pg_parts(total, room, SH_MIN_SHARE);
    const int near = pg_near(total, parts);
    auto holder = [&](int64_t cut) {
      long i = 0;
      for (long x = 0; x < items; ++x)
        if (line[x] <= cut) i = x;
      return i;
    };
    for (int64_t p = 0; p < parts && total > 0; ++p) {
      const int64_t cut[2] = {pg_cut(total, parts, p), pg_cut(total, parts, p + 1)};
      long from[2];
      int tile[2], step[2];
      for (int e = 0; e < 2; ++e) {
        from[e] = streams, tile[e] = step[e] = 0;
        if (cut[e] < line[streams]) {
          from[e] = holder(cut[e]);
          sh_place(cut[e] - line[from[e]], (int)n[from[e]], (int)rows[from[e]], from[e] < groups ? SH_GROUP : SH_OWN, near, &tile[e], &step[e]);
        }
      }
      for (long x = from[0], t0 = tile[0], begin = step[0]; x < streams && x <= from[1]; ++x, t0 = 0, begin = 0)
        for (long t = t0; n[x] > 0 && t * sh_tile((int)rows[x]) < rows[x]; ++t, begin = 0) {
          if (x == from[1] && t > tile[1]) break;
          const long end = x == from[1] && t == tile[1] ? step[1] : n[x];
          if (begin < end) printf("g %ld %ld %ld %ld %ld\\n", (long)p, x, t, begin, end);
        }
      const int64_t own[2] = {cut[0] > line[streams] ? cut[0] : line[streams], cut[1] > line[streams] ? cut[1] : line[streams]};
      for (long w = 0; w < SH_WAVES; ++w) {
        long b[2] = {items, items}, s[2] = {0, 0};
        for (int e = 0; e < 2; ++e) {
          const int64_t c = own[0] + (own[1] - own[0]) * (w + e) / SH_WAVES;
          if (c >= total) continue;
          b[e] = holder(c);
          s[e] = sh_stream_step(c - line[b[e]], (int)n[b[e]]);
        }
        for (long x = b[0], begin = s[0]; x < items && x <= b[1]; ++x, begin = 0) {
          const long end = x == b[1] ? (s[1] < n[x] ? s[1] : n[x]) : n[x];
          if (begin < end) printf("s %ld %ld 0 %ld %ld\\n", (long)(p * SH_WAVES + w), x, begin, end);
        }
      }
    }
    printf("end\\n");
  }
}
"""


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    tmp = tmp_path_factory.mktemp("plan")
    (tmp / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-Wall", "-Werror", "-Wno-unused-function", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC,
                    str(tmp / "plan.cpp"), "-o", str(tmp / "plan")], check=True)

    def run(cases):
        text = "".join(f"{len(items)} {min(streams, len(items) // 2)} {streams} {room} " + " ".join(f"{n} {rows}" for n, rows in items) + "\n" for items, streams, room in cases)
        out = subprocess.run([str(tmp / "plan")], input=text, capture_output=True, text=True, check=True).stdout
        found, here = [], []
        for line in out.splitlines():
            if line == "end":
                found.append(here)
                here = []
            else:
                kind, *rest = line.split()
                here.append((kind, *map(int, rest)))
        return found

    return run


def _tile(rows):
    return 64 if rows <= 64 else 128


@pytest.mark.parametrize("seed", range(6))
def test_every_step_falls_to_one_part(ask, seed):
    rng = random.Random(seed)
    cases = []
    for _ in range(150):
        items = [(rng.choice((0, 1, 2, rng.randrange(1, 40), rng.randrange(1, 2000))), rng.choice((0, 1, 4, 64, 65, 128, 129, rng.randrange(1, 700)))) for _ in range(rng.randrange(1, 30))]
        streams = rng.choice((len(items), 0, rng.randrange(0, len(items) + 1)))
        items = [(n, rows if i < streams else min(max(rows, 1), 16)) for i, (n, rows) in enumerate(items)]
        cases.append((items, streams, rng.choice((1, 2, 32, 64, 256))))
    for (items, streams, room), pieces in zip(cases, ask(cases)):
        parts = {}
        for kind, part, item, tile, begin, end in pieces:
            assert (kind == "s") == (item >= streams) and begin < end
            parts.setdefault((item, tile), []).append((part, begin, end))
        for i, (n, rows) in enumerate(items):
            for tile in range(-(-rows // _tile(rows)) if i < streams else 1):
                got = parts.pop((i, tile), [])
                if n == 0 or rows == 0:
                    assert not got
                    continue
                assert [b for _, b, _ in got] == [0] + [e for _, _, e in got[:-1]] and got[-1][2] == n, (i, tile, got)
                assert [p for p, _, _ in got] == list(range(got[0][0], got[0][0] + len(got)))  # side by side
        assert not parts
        # a part has at most one piece that began in an earlier one, its first, and one that goes on, its last
        of_part = {}
        for kind, part, item, tile, begin, end in pieces:
            of_part.setdefault((kind, part), []).append((begin > 0, end < items[item][0]))
        for edges in of_part.values():
            assert not any(begun for begun, _ in edges[1:]) and not any(on for _, on in edges[:-1])


def test_very_long_lines(ask):
    """Requests of 2^30 keys: units past 31 bits."""
    n = 1 << 25
    items = [(n, 700)] * 20 + [(n, 4)] * 90
    for streams in (20, 110):
        pieces = ask([(items, streams, 32)])[0]
        assert sum(end - begin for kind, _, _, _, begin, end in pieces) == 20 * 6 * n + 90 * n


def test_cuts_in_doubles_are_the_cuts(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    (tmp_path / "cuts.cpp").write_text("""
#include <stdio.h>
#include "sp_paged_plan.h"
int main() {
  uint64_t x = 1;
  long bad = 0;
  for (int i = 0; i < 20000; ++i) {
    x = x * 6364136223846793005ull + 1442695040888963407ull;
    const int parts = 1 + (int)(x >> 40) % 512;
    const int64_t total = (int64_t)((x >> 8) & ((1ull << (1 + i % 36)) - 1)) / (i % 3 ? 1 : parts) * (i % 3 ? 1 : parts);
    const PgCuts cuts = pg_cuts(total, parts);
    for (int p = 0; p <= parts + 1; ++p) bad += pg_cut_at(cuts, p) != (p > parts ? total : (int64_t)((unsigned __int128)total * p / parts));
  }
  const PgCuts cuts = pg_cuts((1ll << 59) + 12345, 511);  // (beyond: in order, from 0 to the end)
  for (int p = 0; p < 511; ++p) bad += pg_cut_at(cuts, p + 1) < pg_cut_at(cuts, p);
  bad += pg_cut_at(cuts, 0) != 0 || pg_cut_at(cuts, 511) != (1ll << 59) + 12345;
  printf("%ld\\n", bad);
}
""")
    subprocess.run(["g++", "-O2", "-Wall", "-I", CSRC, str(tmp_path / "cuts.cpp"), "-o", str(tmp_path / "cuts")], check=True)
    assert subprocess.run([str(tmp_path / "cuts")], capture_output=True, text=True, check=True).stdout.strip() == "0"
