"""What the tiles of a chunk walk behind a window with sinks: the planner's host arithmetic against the blocks counted row by row."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinytitan_amd", "csrc")

PROGRAM = r'''
#include <cstdio>
#include <set>
#include "chunk_plan.h"

static int check(int start, int rows, int valid, int window, int sinks) {
    int longest = 0;
    for (int t = 0; 32 * t < rows; ++t) {
        // a tile walks its sinks' blocks and every block from its first row's window to its last row's own key, each once
        std::set<int> blocks;
        for (int row = 32 * t; row < 32 * t + 32 && row < rows; ++row) {
            const int end = start + row + 1 < valid ? start + row + 1 : valid, lo = start + row + 1 > window ? start + row + 1 - window : 0;
            for (int key = lo; key < end; key += 32) blocks.insert(key / 32);
            blocks.insert((end - 1) / 32);
            if (row == 32 * t)
                for (int key = 0; key < sinks && key / 32 < lo / 32; key += 32) blocks.insert(key / 32);
        }
        const int walked = tt::chunk_tile_blocks(start, rows, valid, window, t, sinks);
        if (walked != (int)blocks.size()) {
            std::printf("%d rows behind %d, window %d, %d sinks: tile %d walks %d, not %d\n", rows, start, window, sinks, t, (int)blocks.size(), walked);
            return 1;
        }
        if (walked > longest) longest = walked;
    }
    const tt::KeyRanges r = tt::plan_window_ranges(256, 256, 16, 2, start, rows, valid, window, sinks);
    const bool covered = r.n_splits < 2 || (long long)r.n_splits * r.split_blocks >= longest;
    if (!covered || tt::longest_tile_blocks(start, rows, valid, window, sinks) != longest || tt::most_tile_blocks(start, rows, valid, window, sinks) < longest) {
        std::printf("%d rows behind %d, window %d, %d sinks: longest %d\n", rows, start, window, sinks, longest);
        return 1;
    }
    return 0;
}

int main() {
    int bad = 0;
    for (int window : {1, 31, 32, 33, 100, 512, 2000, 4096})
        for (int sinks : {0, 1, 4, 32, 33, 300, 5000})
            for (int start : {0, 1, 30, 31, 32, 95, 500, 2001, 4100, 9000})
                for (int rows : {1, 31, 32, 33, 64, 301, 1000}) bad += check(start, rows, start + rows + (rows == 64 ? 40 : 0), window, sinks);
    std::printf("%d\n", bad);
    return bad != 0;
}
'''


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_tiles_walk_their_sinks_and_their_window(tmp_path):
    source, program = tmp_path / "plan.cpp", tmp_path / "plan"
    source.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-I", CSRC, str(source), "-o", str(program)], check=True)
    out = subprocess.run([str(program)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout
