"""CPU checks of the rule that gives an MXFP4 product its kernel (csrc/mx4_plan.hpp,
plain arithmetic, run by a host program)."""
import os
import shutil
import subprocess

import pytest

from mx4_sizes import SIZES

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sushiblas_amd", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include "mx4_plan.hpp"

int main()
{
    const char* names[] = {"Narrow2", "Narrow", "Tile64", "Tile64Groups", "Tile128Stages", "Tile128",
                           "Tile256x192", "Tile192x256", "Tile256", "None"};
    int m, n, k;
    while (scanf("%d %d %d", &m, &n, &k) == 3) puts(names[(int)sbx::mx4_kernel(m, n, k)]);
    return 0;
}
"""


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", f"-I{CSRC}", "-o", str(d / "plan"), str(d / "plan.cpp")], check=True)

    def ask(sizes):
        text = "\n".join("%d %d %d" % s for s in sizes)
        res = subprocess.run([str(d / "plan")], input=text, stdout=subprocess.PIPE, text=True, check=True, timeout=60)
        return res.stdout.split()
    return ask


def test_sizes_reach_their_kernels(kernels):
    assert kernels(SIZES.values()) == list(SIZES)


def test_no_terms_go_by_tiles(kernels):
    """Nothing to add up: a large C is written by tiles, as with few terms."""
    got = kernels([(8192, 8192, 0), (4096, 4100, 0), (1500, 2051, 0)])
    assert all(k.startswith("Tile") for k in got)


def test_tall_results_fit_a_launch(kernels):
    side = 1 << 30
    assert kernels([(side, 20, 32), (20, side, 32), (side, 200, 32)]) != ["None"] * 3
    got = kernels([(side, 20, 32), (20, side, 32), (side, side, 32), (1, side, 32)])
    assert set(got[:2]) <= {"Tile256x192", "Tile192x256", "Tile256"}  # (64's and 128's: 2^32 threads)
    assert got[2:] == ["None", "Narrow2"]
