// Which byte of a matrix's square scales (fp8_format.cuh) a product fetches for a lane.  No CUDA in it, all of it constexpr: the kernel calls it, and a test compiles this file
// by itself and compares what it says with the size of the scales.
#pragma once

namespace tuna {

constexpr int fp8_least(int a, int b) { return a < b ? a : b; }

// A product's operand A has `rows` rows (gated: of both projections) and `blocks` blocks of 128 along its sum; a CTA's share of a tile starts at `row0`, which in a pair's last tile may
// lie behind the last row.  Its rows are of one block or two, gated of as many for each projection: `slot` numbers them, and `kb` is the block of the sum.  `across` (dx): A is the matrix
// read across, whose scales lie [blocks][blocks of rows], and a CTA's 128 rows are one block.  What lies behind the last block of either kind is the last one's: nothing is multiplied with it.
constexpr long long fp8_square_scale(bool across, bool gated, int row0, int slot, int kb, int rows, int blocks)
{
    const int row_blocks = (rows + 127) / 128, first = gated ? (slot >> 1) * (rows / 2) + (row0 >> 1) : row0;
    const int block = fp8_least(first / 128 + (across ? 0 : slot & 1), row_blocks - 1), at = fp8_least(kb, blocks - 1);
    return across ? (long long)at * row_blocks + block : (long long)block * blocks + at;
}

}  // namespace tuna
