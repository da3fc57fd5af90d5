"""How many channels a workgroup of the few tokens' 8-bit products takes, against what all three were measured to take: the header's rule, without a
device."""
import shutil
import subprocess

import pytest

from tinytitan_amd import build

# columns, tokens, channels: us by one tile of 16 channels a workgroup, two and four, on 256 CUs
MEASURED = {
    (2048, 1): {4096: (5.1, 4.7, 6.4), 4352: (5.9, 4.8, 6.5), 4576: (6.0, 4.8, 6.5), 5120: (6.1, 4.9, 6.5), 8192: (6.6, 5.7, 6.9), 8224: (8.3, 8.4, 6.9),
                8704: (8.8, 8.8, 6.9), 9152: (8.9, 8.9, 7.0), 9216: (8.8, 8.9, 7.0), 12288: (9.6, 9.2, 7.6), 16384: (11.8, 10.2, 8.5)},
    (2048, 7): {3584: (4.0, 4.5, 5.9), 4096: (4.1, 4.5, 5.9), 4352: (4.9, 4.6, 6.0), 8192: (5.3, 5.5, 6.4), 8224: (6.9, 8.0, 6.4), 9152: (7.2, 8.5, 6.5), 16384: (9.7, 9.9, 8.5)},
    (2048, 32): {4096: (5.1, 5.8, 8.1), 4352: (8.4, 5.9, 8.3), 8192: (9.0, 6.9, 9.1), 8224: (11.9, 10.3, 8.9), 9152: (12.1, 10.6, 9.0), 16384: (16.9, 11.9, 10.7)},
    (2048, 64): {4096: (6.6, 8.1, 8.4), 4352: (11.0, 8.1, 8.5), 8192: (11.7, 8.7, 8.8), 8224: (15.8, 14.3, 8.8), 12288: (17.0, 15.4, 9.2)},
    (4096, 1): {3584: (5.9, 6.9, 9.1), 4096: (6.4, 7.3, 9.3), 4352: (8.1, 7.3, 9.3), 4576: (8.0, 7.4, 9.4), 8192: (9.6, 9.5, 10.8), 8224: (11.2, 13.5, 10.6),
                9152: (11.8, 13.8, 10.8), 12288: (14.0, 15.1, 12.6), 16384: (16.7, 17.4, 15.5)},
    (4096, 32): {4096: (7.6, 8.5, 11.8), 4352: (11.9, 8.5, 12.0), 8192: (13.7, 10.3, 13.4), 8224: (17.2, 15.3, 13.3), 9152: (17.8, 15.5, 13.6), 16384: (25.2, 19.0, 18.1)},
    (4096, 64): {4096: (9.7, 11.3, 12.8), 4352: (16.0, 11.5, 13.1), 8192: (17.6, 13.2, 14.0), 8224: (23.4, 21.2, 14.1), 12288: (25.5, 22.5, 15.4)},
}


def test_no_measured_product_is_a_tenth_slower_than_by_its_best_tiles(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    (tmp_path / "rule.cpp").write_text('#include <cstdio>\n#include <cstdlib>\n#include "int8_plan.h"\nint main(int n, char **v) {\n'
                                       '    for (int i = 1; i < n; ++i) std::printf("%d\\n", tt::int8_ring_tiles(256, std::atoi(v[i])));\n}\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", build.CSRC, str(tmp_path / "rule.cpp"), "-o", str(tmp_path / "rule")], check=True)

    def tiles(channels):
        return [int(t) for t in subprocess.run([str(tmp_path / "rule"), *map(str, channels)], capture_output=True, text=True, check=True).stdout.split()]

    for (columns, tokens), rows in MEASURED.items():
        for (channels, us), taken in zip(rows.items(), tiles(rows)):
            assert us[{1: 0, 2: 1, 4: 2}[taken]] <= 1.1 * min(us), (columns, tokens, channels, taken)
    assert tiles([1, 16, 4096, 4097, 8192, 8193, 2 ** 31 - 1]) == [1, 1, 1, 2, 2, 4, 4]
