"""The prefix sums that the bookkeeping of a cache in pages forms (csrc/sp_paged_plan.h, arithmetic of the device alone), on the CPU: sums of
whatever the requests' lengths are hold at 2^30, stay sorted, do not depend on the order they are formed in, and a search in them ends at the
request that holds what is asked for."""

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
  int n, m;
  while (scanf("%d %d", &n, &m) == 2) {  // lengths, questions
    std::vector<int> x(n), sums(n + 1);
    for (int& v : x) scanf("%d", &v), v = pg_length(v);
    int at = 0, halves[2] = {0, 0};
    for (int i = 0; i < n; ++i) {
      sums[i] = at;
      at = pg_held_sum(at, x[i]);
      halves[i >= n / 2] = pg_held_sum(halves[i >= n / 2], x[i]);
    }
    sums[n] = at;
    printf("%d", pg_held_sum(halves[0], halves[1]));
    for (int s : sums) printf(" %d", s);
    for (int q; m-- > 0;) scanf("%d", &q), printf(" %d", pg_holder(sums.data(), n, q));
    printf("\\n");
  }
}
"""
HELD = 1 << 30


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    tmp = tmp_path_factory.mktemp("sums")
    (tmp / "sums.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-O1", "-Wall", "-Werror", "-Wno-unused-function", "-Wno-unused-result", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", CSRC, str(tmp / "sums.cpp"), "-o", str(tmp / "sums")], check=True)

    def run(lengths, questions):
        text = "%d %d\n%s\n%s\n" % (len(lengths), len(questions), " ".join(map(str, lengths)), " ".join(map(str, questions)))
        out = subprocess.run([str(tmp / "sums")], input=text, capture_output=True, text=True, check=True).stdout
        values = list(map(int, out.split()))
        return values[0], values[1:len(lengths) + 2], values[len(lengths) + 2:]

    return run


def _cases():
    top = 2 ** 31 - 1
    yield [top] * 4
    yield [top] * 4096
    yield [HELD - 1, 1, HELD - 1, HELD - 1, 5, top, 0, 7]
    yield [5, top, 3, top, top, 2, 0, top, -1, 9]
    yield [HELD // 2, HELD // 2, HELD // 2, 1]
    yield [-2 ** 31, -1, 0, 0]
    yield [3]
    rng = random.Random(4)
    for _ in range(60):
        yield [rng.choice((0, 1, rng.randrange(500), rng.randrange(2 ** 31), top, HELD - 1, -5)) for _ in range(rng.randrange(1, 60))]


def test_sums_hold_and_stay_sorted(ask):
    rng = random.Random(5)
    for lengths in _cases():
        held = [max(0, min(n, HELD - 1)) for n in lengths]
        want = [min(sum(held[:i]), HELD) for i in range(len(held) + 1)]
        below = [x for x in {0, 1, want[-1] - 1, *[w for w in want], *[w - 1 for w in want], rng.randrange(max(want[-1], 1))} if 0 <= x < want[-1]]
        in_halves, sums, holders = ask(lengths, below)
        assert sums == want and in_halves == want[-1]
        for x, b in zip(below, holders):
            assert sums[b] <= x < sums[b + 1], "the request that place x belongs to"
