"""The runs of work that the attention over a cache in pages deals out (csrc/page_runs.hpp), compiled
for the host: every unit's runs against a count step by step, and the runs of a unit whose bounds do
not belong together (lengths that changed during a call), which have to be runs that exist."""
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-30brust_amd", "csrc")

DRIVER = r'''
#include <cstdio>
#include "page_runs.hpp"
int main() {
    unsigned long long total, most, begin, end, units, u;
    while (std::scanf("%llu %llu %llu %llu %llu %llu", &total, &most, &begin, &end, &units, &u) == 6) {
        const qh::Parts p = qh::parts_of(total, most, begin, end, units, u);
        const unsigned long long runs = qh::runs_of(total, most);
        std::printf("%llu %llu %u\n", runs, (unsigned long long)p.first, p.count);
    }
}
'''


@pytest.fixture(scope="module")
def parts(tmp_path_factory):
    where = tmp_path_factory.mktemp("runs")
    (where / "runs.cpp").write_text(DRIVER)
    subprocess.run(["g++", "-O1", "-std=c++17", "-D__host__=", "-D__device__=", "-I", CSRC, str(where / "runs.cpp"), "-o",
                    str(where / "runs")], check=True)

    def ask(rows):
        text = "".join(" ".join(map(str, r)) + "\n" for r in rows)
        out = subprocess.run([str(where / "runs")], input=text, capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return ask


def test_runs_of_units(parts):
    rng, rows, want = random.Random(1), [], []
    for _ in range(300):
        units, most = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 7, 64, 1024])
        steps = [2 + max(1, rng.randint(0, 40) if rng.random() < 0.8 else rng.randint(0, 900)) for _ in range(rng.randint(1, 9))]
        total = units * sum(steps)
        runs = min((total + 1) // 2, most)
        bounds = [total * i // runs for i in range(runs + 1)]
        run_of = [i for i in range(runs) for _ in range(bounds[i], bounds[i + 1])]
        before = 0
        for n in steps:
            for u in range(units):
                held = run_of[before + u * n + 2:before + (u + 1) * n]  # two steps are not work
                rows.append((total, most, before, before + units * n, units, u))
                want.append((runs, held[0], held[-1] - held[0] + 1))
            before += units * n
    assert parts(rows) == want


def test_bounds_that_do_not_belong_together(parts):
    rng, rows = random.Random(2), []
    for _ in range(20000):
        units, most = rng.choice([1, 2, 32, 65535]), rng.choice([1, 5, 1024, 2048])
        total = rng.choice([3, rng.randint(3, 500), rng.randint(3, 1 << 50)])
        begin, end = (rng.choice([0, total, total - 1, rng.randint(0, total), rng.randint(0, (1 << 64) - 1), (1 << 64) - 1])
                      for _ in range(2))
        rows.append((total, most, begin, end, units, rng.randrange(units)))
    for row, (runs, first, count) in zip(rows, parts(rows)):
        assert 1 <= runs <= row[1] and first + count <= runs, row
