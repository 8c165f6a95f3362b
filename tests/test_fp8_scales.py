"""Which bytes of the square scales the 8-bit products fetch: none outside of them, and of the rows and blocks that there are the right ones."""

import subprocess

import pytest

from tuna_b200 import build

PROGRAM = """
#include <cstdio>
#include <cstdlib>
#include "fp8_scales.h"
using tuna::fp8_square_scale;
static long long outside = 0, wrong = 0, seen = 0;
static void see(bool across, bool gated, int row0, int slots, int rows, int red)
{
    const int row_blocks = (rows + 127) / 128, blocks = (red + 127) / 128;
    for (int slot = 0; slot < slots; ++slot)
        for (int kb = 0; kb < (blocks + 15) / 16 * 16; ++kb) {  // groups of four units of up to four blocks
            const long long at = fp8_square_scale(across, gated, row0, slot, kb, rows, blocks);
            ++seen;
            if (at < 0 || at >= (long long)row_blocks * blocks) ++outside;
            // a row of the slot that there is, and a block that there is
            const int half = gated ? (slot >> 1) * (rows / 2) : 0, end = gated ? half + rows / 2 : rows, first = half + (gated ? row0 >> 1 : row0);
            const int row = (slot & 1) ? (first / 128 + 1) * 128 : first;
            if (row < end && kb < blocks && at != (across ? (long long)kb * row_blocks + row / 128 : (long long)(row / 128) * blocks + kb)) ++wrong;
        }
}
int main(int, char **argv)
{
    const int rows = std::atoi(argv[2]), red = std::atoi(argv[3]);
    if (argv[1][0] == 'x') {  // dx: pairs of 128 rows
        for (int b = 0; b < 2 * ((rows + 255) / 256); ++b) see(true, false, 128 * b, 1, rows, red);
    } else {
        const bool gated = argv[1][0] == 'g';
        const int slots = gated ? 4 : 2;
        for (int b = 0; b < 2 * ((rows + 255) / 256); ++b) see(false, gated, 128 * b, slots, rows, red);
        for (int row0 = 0; row0 < rows; row0 += 4) see(false, gated, row0, slots, rows, red);  // single CTAs: tiles of any height
    }
    std::printf("%lld %lld %lld\\n", outside, wrong, seen);
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("fp8_scales")
    (d / "scales.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{build.CSRC}", str(d / "scales.cpp"), "-o", str(d / "scales")], check=True)
    return str(d / "scales")


# rows of A (in dx the matrix's columns) of odd and even numbers of blocks, whole and not
@pytest.mark.parametrize("rows", [16, 112, 128, 144, 256, 272, 384, 400, 512, 528, 784, 1040, 1360, 2720, 4096, 4112])
@pytest.mark.parametrize("red", [16, 128, 144, 256, 1040, 1552, 2720, 65536])
@pytest.mark.parametrize("form", ["product", "gated", "x"])
def test_no_scale_outside_is_read(program, form, rows, red):
    if form == "gated" and rows % 32:
        rows += 16  # two projections of a multiple of 16 features
    outside, wrong, seen = map(int, subprocess.run([program, form, str(rows), str(red)], check=True, capture_output=True, text=True).stdout.split())
    assert seen and not outside and not wrong
