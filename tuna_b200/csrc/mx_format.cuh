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

// Numbers are read once and kept out of L1, by a coherent load: the kernels that quantize a product's tokens are resident while the kernel
// that writes these may still run, and the read-only path (ld.global.nc) is for memory that nobody writes as long as the reading kernel lives.
__device__ __forceinline__ uint4 mx_load_u4(const void *p)
{
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.L2::128B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

// Eight numbers of type T as they lie in memory, their largest magnitude and their values.
template <typename T>
struct Mx8;
template <>
struct Mx8<__half> {
    uint4 r;
    __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const __half *p) { r = mx_load_u4(p); }
    __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }
    __device__ __forceinline__ __half2 pair(int i) const { const uint32_t w = word(i); return *reinterpret_cast<const __half2 *>(&w); }
    // Bits (fp32) of the largest magnitude of the four lanes' 32 numbers; NaN's if there is one.
    __device__ __forceinline__ uint32_t largest() const
    {
        __half2 m = __hmax2_nan(__hmax2_nan(__habs2(pair(0)), __habs2(pair(1))), __hmax2_nan(__habs2(pair(2)), __habs2(pair(3))));
        m = __hmax2_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = __hmax2_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
        return __float_as_uint(__half2float(__hmax_nan(__low2half(m), __high2half(m)))) & 0x7fffffffu;
    }
    __device__ __forceinline__ void values(float (&v)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(pair(i));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};
template <>
struct Mx8<__nv_bfloat16> {
    uint4 r;
    __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { r = mx_load_u4(p); }
    __device__ __forceinline__ uint32_t word(int i) const { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }
    __device__ __forceinline__ __nv_bfloat162 pair(int i) const { const uint32_t w = word(i); return *reinterpret_cast<const __nv_bfloat162 *>(&w); }
    __device__ __forceinline__ uint32_t largest() const
    {
        __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(__habs2(pair(0)), __habs2(pair(1))), __hmax2_nan(__habs2(pair(2)), __habs2(pair(3))));
        m = __hmax2_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = __hmax2_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
        return ((uint32_t)__bfloat16_as_ushort(__hmax_nan(__low2bfloat16(m), __high2bfloat16(m))) & 0x7fffu) << 16;
    }
    __device__ __forceinline__ void values(float (&v)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(word(i) << 16);
            v[2 * i + 1] = __uint_as_float(word(i) & 0xffff0000u);
        }
    }
};
template <>
struct Mx8<float> {
    uint4 r, t;
    __device__ __forceinline__ void zero() { r = t = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const float *p) { r = mx_load_u4(p); t = mx_load_u4(p + 4); }
    __device__ __forceinline__ uint32_t largest() const
    {
        const uint32_t w[8] = {r.x, r.y, r.z, r.w, t.x, t.y, t.z, t.w};
        uint32_t m = 0;  // magnitudes compare as their bits do, NaN above infinity
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7fffffffu);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    }
    __device__ __forceinline__ void values(float (&v)[8]) const
    {
        const uint32_t w[8] = {r.x, r.y, r.z, r.w, t.x, t.y, t.z, t.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    }
};

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
