// The microscaled 4-bit format (OCP MXFP4) on the device: e2m1 codes, one e8m0 scale (exponent + 127; 255 is NaN) for every 32
// columns of a row.  Layout: codes in chunks of 256 columns, [chunk][row][128 bytes], column 2j of a chunk in the low nibble of
// byte j, 2j+1 in the high one; scales in 32-bit words of four, [128 columns][row][4 bytes].  So the rows of a tile, whatever
// row it starts at, are one run of memory for every chunk: 16 KB of codes and two of 512 bytes of scales for 128 rows.
#pragma once
#include <cuda_bf16.h>
#include "common.cuh"

namespace tuna {

constexpr int kMxBlock = 32;       // columns that share a scale
constexpr int kMxChunk = 256;      // columns of a chunk of codes: 128 bytes, one row of a swizzled shared-memory tile
constexpr int kMxScaleCols = 128;  // columns of a word of scales
constexpr int kMxChunkBytes = kMxChunk / 2;

// Eight numbers of type T from 16 (32) bytes, as fp32.
__device__ __forceinline__ void mx_load8(const __half *p, float (&v)[8])
{
    const uint4 r = ldg_stream_u4(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void mx_load8(const __nv_bfloat16 *p, float (&v)[8])
{
    const uint4 r = ldg_stream_u4(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void mx_load8(const float *p, float (&v)[8])
{
    const uint4 a = ldg_stream_u4(p), b = ldg_stream_u4(p + 4);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}

// The scale of a block whose largest magnitude has the bits `largest` (fp32): floor(log2(largest)) - 2, so that the largest
// lies between 4 and 8 times the scale (what is above 6 saturates), not below 2^-127.  Infinity or NaN: a NaN scale.
__device__ __forceinline__ uint32_t mx_scale(uint32_t largest)
{
    const int e = (int)(largest >> 23) - 2;  // a subnormal's field is 0, as that of zero
    return largest >= 0x7f800000u ? 255u : (uint32_t)max(e, 0);
}
// 1 / scale for the scales that mx_scale gives (0 .. 252): a power of two, so the product is exact where it matters.
__device__ __forceinline__ float mx_inverse(uint32_t s) { return __uint_as_float((254u - min(s, 252u)) << 23); }
// 2^(s - 127); NaN for 255.
__device__ __forceinline__ float mx_scale_value(uint32_t s)
{
    return __uint_as_float(s == 255u ? 0x7fffffffu : s == 0u ? 0x00400000u : s << 23);
}

// Eight numbers -> eight codes, the first in the lowest nibble: to the nearest, ties to even, saturating at 6.
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8])
{
    uint32_t d;
    asm("{\n .reg .b8 a, b, c, d;\n"
        " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        " mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(d)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return d;
}
// Eight codes -> eight numbers as four pairs of fp16 (exact).
__device__ __forceinline__ void mx_decode8(uint32_t w, uint32_t (&h)[4])
{
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
        " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}

}  // namespace tuna
