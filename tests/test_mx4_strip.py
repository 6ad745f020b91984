"""CPU check of where the MXFP4 product's narrow kernel reads (csrc/mx4_strip.hpp):
no load that passes the range check of its vector offset, which is the one part
that is certain to be tested, reads past the operand's end, also where the strip
has few rows or the last group few blocks; and what is inside is read.

The header is plain arithmetic; a host program runs it over strips of every row
count, over ragged block counts and padded rows."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sushiblas_amd", "csrc")

PROGRAM = r"""
#include <stdio.h>
#include <initializer_list>
#include "mx4_strip.hpp"
using namespace sbx;

static int check(int rows, int ld, int blocks, long& loads)
{
    const unsigned bytes = (unsigned)strip_bytes(rows, ld, blocks);
    const int groups = (blocks + 7) / 8;
    for (int i = 0; i < N; ++i)
        for (int g = 0; g < groups + 16; ++g)  // the kernel asks for groups past the last one too
            for (int lane = 0; lane < 64; ++lane)
                for (int half = 0; half < 2; ++half) {
                    const int left = blocks - 8 * g;
                    const unsigned v = (unsigned)strip_vector(strip_lane(lane, i, rows, ld), lane, half, left);
                    const unsigned s = (unsigned)strip_scalar(i, g, rows, ld, left);
                    const int row = 16 * i + lane % 16, block = 8 * g + lane / 16 * 2 + half;
                    const bool inside = row < rows && block < blocks, read = v < bytes;
                    // the scalar offset is never past the end, were it taken from the size instead
                    const bool right = inside ? (unsigned long long)v + s == (unsigned long long)row * ld + 16ull * block
                                              : v >= 0x80000000u;
                    if (read != inside || !right || s > bytes || (read && (unsigned long long)v + s + 16 > bytes)) {
                        printf("N %d rows %d ld %d blocks %d: i %d g %d lane %d half %d: %u + %u of %u\n", N, rows, ld,
                               blocks, i, g, lane, half, v, s, bytes);
                        return 1;
                    }
                    loads += read;
                }
    return 0;
}

int main()
{
    long loads = 0;
    for (int rows = 1; rows <= 16 * N; ++rows)
        for (int blocks : {1, 2, 3, 7, 8, 9, 15, 16, 17, 63, 64, 219})
            for (int pad : {0, 16, 4096})
                if (check(rows, 16 * blocks + pad, blocks, loads)) return 1;
    // the longest rows that the entry point takes
    if (check(16 * N, (1 << 23) - 16, 9, loads) || check(1, (1 << 23) - 16, 3, loads)) return 1;
    printf("%ld loads inside\n", loads);
    return 0;
}
"""


@pytest.mark.parametrize("n", [1, 2])
def test_strip_loads_stay_inside(tmp_path, n):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    src, exe = tmp_path / "strip.cpp", tmp_path / "strip"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++17", "-O1", f"-DN={n}", f"-I{CSRC}", "-o", str(exe), str(src)], check=True)
    res = subprocess.run([str(exe)], stdout=subprocess.PIPE, text=True, timeout=100)
    assert res.returncode == 0, res.stdout
    assert int(res.stdout.split()[0]) > 0
