"""How attention over pages and windows is cut into work (csrc/sp_paged_plan.h, arithmetic that host and device share), on the CPU: the units
that a row tile walks hold every key that one of its rows sees, row tiles number without a clash, and the cuts of a line cover it once."""

import os
import random
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "shareprefill_amd", "csrc")
PROGRAM = """
#include <stdio.h>
#include "sp_paged_plan.h"
int main() {
  char what;
  long a, b, c, d, e;
  while (scanf(" %c %ld %ld %ld %ld %ld", &what, &a, &b, &c, &d, &e) == 6) {
    if (what == 's') {
      const PgSpan s = pg_span((int)a, (int)b, (int)c, (int)d, (int)e);
      printf("%d %d %d %d\\n", s.front, s.lo, s.hi, pg_span_units(s));
    } else if (what == 'f') {
      printf("%ld %ld %ld\\n", (long)pg_first_slot(a, (int)b, (int)c, (int)d), (long)pg_slots(a, (int)b, (int)c, (int)d), (long)pg_row_tiles(a, (int)b, (int)d));
    } else if (what == 'c') {
      printf("%ld %ld\\n", (long)pg_parts(a, b, 3), (long)pg_cut(a, pg_parts(a, b, 3), c));
    } else if (what == 'n') {
      printf("%d %d\\n", pg_snap(a, (int)b, 2, pg_near(c, d)), pg_near(c, d));
    } else if (what == 'q') {
      printf("%u\\n", pg_div((unsigned)a, pg_divisor((unsigned)b)));
    } else if (what == 'd') {
      const long part = b;
      int seq = -1, rt = -1;
      const bool any = pg_deal((int)a, (int)part, (int)c, (int)d, (int)e, pg_together((int)e, (int)c, (int)d), &seq, &rt);
      printf("%d %d %d\\n", any ? 1 : 0, seq, rt);
    } else {
      int p0, p1;
      pg_tile_positions((int)a, (int)b, (int)c, pg_divisor((unsigned)d), (int)e, &p0, &p1);
      printf("%d %d\\n", p0, p1);
    }
  }
}
"""
NONE = 1 << 30  # PG_NO_WINDOW


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    tmp = tmp_path_factory.mktemp("plan")
    (tmp / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-Wall", "-Werror", "-Wno-unused-function", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC,
                    str(tmp / "plan.cpp"), "-o", str(tmp / "plan")], check=True)

    def run(questions):
        text = "".join("%s %d %d %d %d %d\n" % (q + (0,) * (6 - len(q))) for q in questions)
        out = subprocess.run([str(tmp / "plan")], input=text, capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return run


@pytest.mark.parametrize("unit", [32, 64])
def test_spans_hold_every_key_that_is_seen_and_no_unit_twice(ask, unit):
    rng = random.Random(unit)
    cases = [(-5, -1, NONE, 0), (-3, 2, 5, 1), (0, 0, 1, 0), (2 ** 30 - 1, 2 ** 30 - 1, NONE, NONE), (-2 ** 30, -2 ** 30, NONE, NONE)]
    for _ in range(400):
        p0 = rng.randrange(-20, 700)
        cases.append((p0, p0 + rng.randrange(0, 130), rng.choice((NONE, rng.randrange(1, 600))), rng.choice((0, 4, rng.randrange(0, 500), NONE))))
    for (p0, p1, window, sinks), (front, lo, hi, n) in zip(cases, ask([("s", *c, unit) for c in cases])):
        assert 0 <= front <= lo and (lo <= hi or hi == 0) and n == front + hi - lo and n >= 0
        if p1 > 1000:
            assert hi == p1 // unit + 1
            continue
        units = list(range(front)) + list(range(lo, hi))
        seen = {j // unit for p in range(p0, p1 + 1) for j in range(max(p, -1) + 1) if j > p - window or j < sinks}
        assert seen <= set(units), (p0, p1, window, sinks)
        # a unit that nobody sees anything of is walked nowhere but between the first sink and the first window's start
        assert all(u in seen for u in units), (p0, p1, window, sinks)


@pytest.mark.parametrize("tile", [128, 256])
def test_row_tiles_number_without_a_clash(ask, tile):
    rng = random.Random(1)
    for _ in range(60):
        g, lens = rng.choice((1, 4, 7, 8, 20, 160)), [rng.choice((0, 1, 2, rng.randrange(300))) for _ in range(rng.randrange(1, 40))]
        at = [0]
        for n in lens:
            at.append(at[-1] + n)
        firsts = [r[0] for r in ask([("f", s, g, b, tile) for b, s in enumerate(at)])]
        tiles = [r[2] for r in ask([("f", n, g, 0, tile) for n in lens])]
        slots = ask([("f", at[-1], g, len(lens), tile)])[0][1]
        for b, n in enumerate(lens):
            assert tiles[b] == -(-n * g // tile)
            assert firsts[b] + tiles[b] <= firsts[b + 1], "room for the tiles of every sequence"
            assert firsts[b] < firsts[b + 1]
        assert firsts[-1] == slots
        # positions of a tile's rows
        b = rng.randrange(len(lens))
        for rt in range(tiles[b]):
            rows = range(rt * tile, min(rt * tile + tile, lens[b] * g))
            assert ask([("p", rt, lens[b], 1000, g, tile)])[0] == (1000 - lens[b] + rows[0] // g, 1000 - lens[b] + rows[-1] // g)


def test_cuts_cover_the_line_once(ask):
    rng = random.Random(2)
    for _ in range(200):
        tiles = [rng.choice((0, 1, 3, 8, rng.randrange(1, 2000))) for _ in range(rng.randrange(1, 30))]
        room = rng.choice((1, 2, 12, 64, 512))
        starts = [0]
        for n in tiles:
            starts.append(starts[-1] + n + 2)
        total = starts[-1]
        parts = ask([("c", total, room, 0)])[0][0]
        assert 1 <= parts <= room
        cuts = [r[1] for r in ask([("c", total, room, p) for p in range(parts + 1)])]
        assert cuts[0] == 0 and cuts[-1] == total and all(a < b for a, b in zip(cuts, cuts[1:]))
        places = []
        for cut in cuts:
            if cut == total:
                places.append((len(tiles), 0))
                continue
            x = max(i for i, s in enumerate(starts[:-1]) if s <= cut)
            tile, near = ask([("n", cut - starts[x], tiles[x], total, parts)])[0]
            assert 0 <= tile <= tiles[x]
            places.append((x, tile) if tile < tiles[x] or tile == 0 else (x + 1, 0))
        assert places[0] == (0, 0) and places == sorted(places)
        # no cut lies within a quarter of a part of a row tile's start or end, four blocks at most
        near = max(1, min(4, total // parts // 4))
        for x, t in places:
            assert t == 0 or near <= t <= tiles[x] - near


def test_a_line_past_32_bits_is_cut_evenly(ask):
    total, parts = 2 ** 45 + 12345, 512
    cuts = [r[1] for r in ask([("c", total, parts, p) for p in range(parts + 1)])]
    assert cuts[-1] == total and all(abs((b - a) - total / parts) < 1.5 for a, b in zip(cuts, cuts[1:]))


def test_whole_row_tiles_are_dealt_once_and_evenly(ask):
    for workgroups, batch, tiles in ((1, 1, 1), (32, 1, 5), (32, 8, 16), (64, 3, 100), (256, 40, 7), (5, 11, 13), (32, 1, 128), (7, 2048, 1)):
        turns = -(-batch * tiles // workgroups)
        asked = [("d", t, p, workgroups, batch, tiles) for t in range(turns) for p in range(workgroups)]
        answers = ask(asked)
        dealt = [(b, rt) for there, b, rt in answers if there]
        assert sorted(dealt) == [(b, rt) for b in range(batch) for rt in range(tiles)]
        # all but the last turn give every workgroup one, and the tiles of a deal of sequences come longest first
        assert all(there for there, _, _ in answers[:(turns - 1) * workgroups])
        if batch == 1:
            assert [max(rt for there, _, rt in answers[t * workgroups:(t + 1) * workgroups] if there) for t in range(turns)] == \
                [tiles - 1 - t * workgroups for t in range(turns)]


def test_quotients_by_a_multiplier(ask):
    rng = random.Random(3)
    top = 2 ** 31 - 1
    pairs = [(x, by) for by in list(range(1, 70)) + [127, 128, 129, 1000, 65535, 65536, 65537, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, top]
             for x in (0, 1, by - 1, by, by + 1, top, top - 1, top // by * by, top // by * by - 1, rng.randrange(top)) if 0 <= x <= top]
    pairs += [(rng.randrange(2 ** rng.randrange(1, 32)), rng.randrange(1, 2 ** rng.randrange(1, 31) + 1)) for _ in range(20000)]
    assert [x for x, in ask([("q", x, by) for x, by in pairs])] == [x // by for x, by in pairs]
