"""Up to how many keys differential attention goes in one split, against what both sides were measured to take: the header's rule, without a device."""
import shutil
import subprocess

import pytest

from tinytitan_amd import build

# head dim, bits, keys, us in several splits, us in one: a layer of 48 in turn, 1 to 16 sequences of 32/8 heads of 128, 16/4 of 64, 16/2 of 256
MEASURED = [
    (128, 16, 448, 8.7, 6.1), (128, 16, 640, 8.5, 7.1), (128, 16, 704, 9.0, 7.5), (128, 16, 768, 8.7, 8.1),
    (128, 16, 448, 8.7, 8.0), (128, 16, 576, 9.1, 9.2), (128, 16, 640, 9.2, 9.9), (128, 16, 704, 9.4, 10.4), (128, 16, 768, 9.5, 11.1),
    (128, 16, 640, 10.4, 10.2), (128, 16, 704, 10.6, 10.7), (128, 16, 768, 10.7, 11.5), (128, 16, 640, 13.3, 11.1), (128, 16, 704, 13.6, 11.7), (128, 16, 768, 14.2, 12.5),
    (64, 16, 512, 7.4, 5.1), (64, 16, 1024, 7.6, 7.1), (64, 16, 896, 8.7, 7.4), (64, 16, 1024, 8.0, 8.2), (64, 16, 1024, 9.5, 8.8),
    (256, 16, 448, 9.5, 9.4), (256, 16, 512, 9.5, 10.0), (256, 16, 640, 9.7, 11.2), (256, 16, 448, 10.9, 12.2), (256, 16, 640, 11.2, 16.2), (256, 16, 448, 12.2, 14.0),
    (256, 16, 512, 12.1, 15.2), (256, 16, 640, 12.3, 17.6),
    (128, 8, 512, 8.3, 7.5), (128, 8, 512, 10.2, 8.2), (128, 4, 512, 8.8, 8.1), (128, 4, 512, 10.1, 8.8), (64, 8, 512, 9.8, 6.3), (64, 4, 512, 7.9, 6.5)]


def test_no_measured_length_takes_a_side_that_is_an_eighth_slower_than_the_other_or_more_but_one(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    (tmp_path / "rule.cpp").write_text('#include <cstdio>\n#include "splitk_plan.h"\nint main() {\n    for (int dim : {64, 128, 256})\n'
                                       '        for (int bits : {16, 8, 4}) std::printf("%d %d %d\\n", dim, bits, tt::maps_one_split_up_to(dim, bits));\n}\n')
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-I", build.CSRC, str(tmp_path / "rule.cpp"), "-o", str(tmp_path / "rule")], check=True)
    up_to = {(int(dim), int(bits)): int(keys) for dim, bits, keys in
             (line.split() for line in subprocess.run([str(tmp_path / "rule")], capture_output=True, text=True, check=True).stdout.splitlines())}
    lost = []
    for dim, bits, keys, several, one in MEASURED:
        taken = one if keys <= max(up_to[dim, bits], 384) else several
        if taken > 1.125 * min(several, one):
            lost.append((dim, bits, keys, several, one))
    assert lost == [(128, 16, 768, 14.2, 12.5)], lost
