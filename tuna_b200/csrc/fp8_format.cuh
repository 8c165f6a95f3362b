// The 8-bit block-scaled format on the device: e4m3 codes, row by row, and one e8m0 scale (exponent + 127; 255 is NaN) for every block
// of 128.  Blocks are 128 columns of a row (kFp8Row), 128 rows of a column (kFp8Column) or 128 x 128 (kFp8Square).  The first two are
// what the two products of a step want along the dimension that they sum over, and have their scale bytes in 32-bit words of four blocks:
// row [ceil(k / 512)][rows][4], column [ceil(rows / 512)][k][4].  Square scales are [ceil(rows / 128)][ceil(k / 128)].
#pragma once
#include "launchers.h"
#include "mx_format.cuh"
#include "fp8_gate.cuh"

namespace tuna {

constexpr int kFp8Block = 128;
constexpr int kFp8Word = 4 * kFp8Block;  // what a word of scales covers

// The scale of a block whose largest magnitude has the bits `largest` (fp32): the smallest power of two over which it is not above 448 =
// 1.75 * 2^8, not below 2^-127.  Infinity or NaN: a NaN scale.
__device__ __forceinline__ uint32_t fp8_scale(uint32_t largest)
{
    const int e = (int)(largest >> 23) - 8 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0);  // a subnormal's field is 0, as that of zero
    return largest >= 0x7f800000u ? 255u : (uint32_t)max(e, 0);
}
// 1 / scale for the scales that fp8_scale gives (0 .. 247): a power of two, so the product is exact where it matters.
__device__ __forceinline__ float fp8_inverse(uint32_t s) { return __uint_as_float((254u - min(s, 247u)) << 23); }

// Four numbers -> four codes, the first in the lowest byte: to the nearest, ties to even.
__device__ __forceinline__ uint32_t fp8_encode4(float a, float b, float c, float d)
{
    uint32_t w;
    asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n mov.b32 %0, {l, h};\n}"
        : "=r"(w)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return w;
}
// Four codes -> two pairs of fp16 (exact).
__device__ __forceinline__ void fp8_decode4(uint32_t w, uint32_t (&h)[2])
{
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}" : "=r"(h[0]), "=r"(h[1]) : "r"(w));
}

}  // namespace tuna
