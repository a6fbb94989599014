"""What the launchers do once per device: the class they use, compiled for the host, and that no launcher sets a kernel's
attributes by itself."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "a100-vision-infer_amd", "csrc")

PROGRAM = r"""
#include <cstdio>
#include "per_device.hpp"
int main() {
    fp8lin::OncePerDevice once;
    int acted[70] = {}, bad = 0;
    auto on = [&](int d, int result) { return once(d, [&] { ++acted[d < 0 ? 69 : d]; return result; }); };
    bad |= on(0, 0) != 0 || on(0, 7) != 0 || acted[0] != 1;                    // done once
    bad |= on(1, 5) != 5 || on(1, 5) != 5 || on(1, 0) != 0 || on(1, 5) != 0 || acted[1] != 3;  // tried again while it fails
    bad |= on(63, 0) != 0 || on(63, 1) != 0 || acted[63] != 1;
    bad |= on(64, 0) != 0 || on(64, 3) != 3 || acted[64] != 2 || on(-1, 2) != 2;  // past what is kept: every time
    bad |= on(0, 9) != 0 || acted[0] != 1;
    std::puts(bad ? "bad" : "good");
}
"""


def test_once_per_device(tmp_path):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if not cxx:
        pytest.skip("no host compiler")
    (tmp_path / "t.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-I", CSRC, str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    assert subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout == "good\n"


def test_kernel_attributes_are_set_through_it():
    places = []
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            places += [(name, line.strip()) for line in f if re.search(r"hipFuncSetAttribute|static const hipError_t", line)]
    assert len(places) == 1 and places[0][0] == "device.hpp", places
