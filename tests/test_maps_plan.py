"""How a chunk of differential attention is cut: the header's rule, run over many shapes without a device.  The ranges have to hold every
block of every tile as the kernel walks them, and the partial results have to stay within their bound."""
import os
import shutil
import subprocess

import pytest

from tests.maps_routes import ROUTES
from tinytitan_amd import build

PROGRAM = r'''
#include <cstdio>
#include <cstdlib>
#include "chunk_plan.h"
using namespace tt;
static int check(int cus, int D, int H, int KH, int start, int rows, int window, int bits) {
    const MapsPlan p = plan_maps_chunk(cus, D, H, KH, start, rows, window, bits);
    if (p.n_splits == 0) return p.split_blocks != 0;
    const int group = H / KH, span = 128 / (group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1), tiles = (rows + span - 1) / span;
    long long longest = 0;
    for (int t0 = 0; t0 < rows; t0 += span) {
        const long long end = (long long)start + std::min(rows, t0 + span);
        const long long first = window > 0 && start + t0 + 1LL > window ? start + t0 + 1LL - window : 0;
        longest = std::max(longest, (end + 31) / 32 - first / 32);
    }
    int bad = p.n_splits < 1 || p.n_splits > 32 || p.split_blocks < 1 || (long long)p.n_splits * p.split_blocks < longest;
    if (p.n_splits > 1) bad |= 2LL * H * tiles * span * p.n_splits > kMapsRangeRows || p.split_blocks < 4;
    if (bad) std::printf("cus %d D %d H %d/%d start %d rows %d window %d bits %d: %d x %d of %lld\n", cus, D, H, KH, start, rows, window, bits, p.n_splits, p.split_blocks, longest);
    return bad;
}
int main(int n, char **v) {
    if (n > 1) {
        const MapsPlan p = plan_maps_chunk(256, atoi(v[3]), atoi(v[1]), atoi(v[2]), atoi(v[6]), atoi(v[5]), atoi(v[7]), atoi(v[4]));
        std::printf("%d\n", p.n_splits);
        return 0;
    }
    int bad = 0;
    const int heads[][2] = {{1, 1}, {3, 1}, {6, 3}, {12, 4}, {16, 2}, {32, 8}, {24, 24}, {34, 2}, {128, 8}};
    for (auto &h : heads)
        for (int D : {64, 128, 256})
            for (int bits : {16, 8})
                for (int cus : {256, 64})
                    for (int rows : {1, 2, 31, 33, 64, 127, 129, 333, 777, 1500, 4097, 20000})
                        for (int start : {0, 1, 31, 33, 500, 2047, 9001, 131071, 1000000})
                            for (int window : {0, 1, 31, 32, 33, 500, 4096, 100000}) bad += check(cus, D, h[0], h[1], start, rows, window, bits);
    bad += check(256, 256, 16, 2, 2147483647 - 4097, 4096, 0, 16) + check(256, 64, 16, 2, 2147483647 - 4097, 4096, 2147483647, 16);
    return bad != 0;
}
'''


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    folder = tmp_path_factory.mktemp("plan")
    (folder / "plan.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", build.CSRC,
                    str(folder / "plan.cpp"), "-o", str(folder / "plan")], check=True)
    return str(folder / "plan")


def test_ranges_hold_every_tile(program):
    ran = subprocess.run([program], capture_output=True, text=True)
    assert ran.returncode == 0, ran.stdout[-4000:] + ran.stderr[-2000:]


@pytest.mark.parametrize("H,KH,D,bits,rows,start,window,ring,way", ROUTES)
def test_every_way_is_among_the_measured_chunks(program, H, KH, D, bits, rows, start, window, ring, way):
    splits = int(subprocess.run([program, *map(str, (H, KH, D, bits, rows, start, window))], capture_output=True, text=True, check=True).stdout)
    assert min(splits, 2) == way, splits
