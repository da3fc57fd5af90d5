"""Which way a call of sequences that share a prefix goes: the planner's host arithmetic, compiled here and run over calls."""
import os
import shutil
import subprocess

import pytest

from tests.shared_ways import CASES, ONE_PASS, RANGES, starts

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinytitan_amd", "csrc")

PROGRAM = r'''
#include <cstdio>
#include <vector>
#include "shared_plan.h"
int main() {
    int D, H, KH, bits, rows, front, chunk_kernel, n;
    while (std::scanf("%d %d %d %d %d %d %d %d", &D, &H, &KH, &bits, &rows, &front, &chunk_kernel, &n) == 8) {
        std::vector<int> totals(n);
        for (int &t : totals)
            if (std::scanf("%d", &t) != 1) return 2;
        const int at_once = tt::shared_seqs_at_once(n, rows);
        tt::SharedPlan p;
        if (tt::plan_shared({256, 0, at_once, totals.data(), rows, front, H, KH, D, bits, chunk_kernel != 0}, &p) != TT_HIP_OK) return 3;
        // at once, the ways, ranges and their blocks, the pair's splits: their length and whether they cover the keys of both pieces
        const long long covered = (long long)p.ranges.n_splits * p.ranges.split_blocks * 32;
        std::printf("%d %d %d %d %d %d\n", at_once, (int)p.way, (int)p.without_ranges, p.ranges.n_splits, covered >= front, p.pair.len);
    }
}
'''


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    where = tmp_path_factory.mktemp("plan")
    source, program = where / "plan.cpp", where / "plan"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-I", CSRC, str(source), "-o", str(program)], check=True)

    def run(calls):
        lines = [" ".join(map(str, (D, H, KH, bits, rows, front, int(chunk_kernel), len(totals), *totals)))
                 for H, KH, D, bits, rows, front, chunk_kernel, totals in calls]
        out = subprocess.run([str(program)], input="\n".join(lines), capture_output=True, text=True, check=True)
        return [tuple(map(int, line.split())) for line in out.stdout.splitlines()]

    return run


def _call(case, chunk_kernel=True):
    H, KH, D, bits, prefix, n, rows, _ = case
    return H, KH, D, bits, rows, prefix // 32 * 32, chunk_kernel, [p + rows for p in starts(prefix, n)]


def test_the_calls_whose_values_are_checked_go_every_way(plan):
    got = plan([_call(c) for c in CASES])
    assert {(c[-1], c[3]) for c in CASES} == {(way, bits) for way in range(4) for bits in (16, 8, 4)}  # every way over every precision
    for case, (at_once, way, without, n_splits, covered, _) in zip(CASES, got):
        assert at_once == case[5] and way == case[-1], (case, way)
        assert way != RANGES or (n_splits >= 2 and covered), case
        assert without != RANGES
    # rows that the chunk kernel does not take
    for case, with_it, (_, way, without, *_) in zip(CASES, got, plan([_call(c, False) for c in CASES])):
        assert way == without == with_it[2], case


def test_what_is_served_at_a_time(plan):
    calls = [(16, 2, 256, 16, rows, 2048, True, [2048 + rows + i for i in range(n)]) for n, rows in
             ((1, 1), (1, 5000), (2, 512), (2, 513), (64, 16), (65, 1), (100, 17), (3, 1024), (7, 300))]
    got = plan(calls)
    assert [g[0] for g in got] == [1, 1, 2, 1, 64, 64, 60, 1, 3]
    assert all(g[1] == ONE_PASS for g in got if g[0] == 1)


def test_one_launch_where_the_keys_are_few(plan):
    assert all(g[1] == ONE_PASS for g in plan([(16, 2, 256, bits, 1, 352, True, [352 + 1 + i % 32 for i in range(64)]) for bits in (16, 8, 4)]))
