// The 8-bit block-scaled format on the device: e4m3 codes, row by row, and one e8m0 scale (exponent + 127; 255 is NaN) for every block
// of 128.  Blocks are 128 columns of a row (kFp8Row), 128 rows of a column (kFp8Column) or 128 x 128 (kFp8Square).  The first two are
// what the two products of a step want along the dimension that they sum over, and have their scale bytes in 32-bit words of four blocks:
// row [ceil(k / 512)][rows][4], column [ceil(rows / 512)][k][4].  Square scales are [ceil(rows / 128)][ceil(k / 128)].
#pragma once
#include "launchers.h"
#include "mx_format.cuh"

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

// The activation is g * sigma(p(g)), sigma the logistic function: p = g (SiLU) or 2 sqrt(2 / pi) (g + 0.044715 g^3) (GELU in its tanh form, as
// (1 + tanh(y)) / 2 = sigma(2 y)).
constexpr float kGeluA = 1.5957691216057308f, kGeluB = 0.044715f, kGeluB3 = 0.134145f;  // the last: three times the one before
template <bool GELU>
__device__ __forceinline__ float fp8_gate(float g)
{
    const float p = GELU ? kGeluA * fmaf(kGeluB * g * g, g, g) : g;
    return __fdividef(1.0f, 1.0f + __expf(-p));  // exp overflows to infinity, and the quotient is 0 then
}
// Two numbers, and what one instruction does to both, rounded to nearest.
struct Fp8Two {
    uint64_t v;
    __device__ __forceinline__ Fp8Two() {}
    __device__ __forceinline__ Fp8Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
    __device__ __forceinline__ explicit Fp8Two(float a) : Fp8Two(a, a) {}
    __device__ __forceinline__ float2 both() const
    {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
};
__device__ __forceinline__ Fp8Two operator+(Fp8Two a, Fp8Two b)
{
    Fp8Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Fp8Two fp8_fma(Fp8Two a, Fp8Two b, Fp8Two c)
{
    Fp8Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Fp8Two operator*(Fp8Two a, Fp8Two b)
{
    Fp8Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
// The product of what is to be added to something.  A product of two at once is made one step with a sum that follows by the compiler, although both say that they round; so it is
// the sum with a -0 that the compiler cannot know for one (gradients of 1360 features and 333 tokens 22.0 us; 22.9 with two single products, which it leaves apart and which are as fast for SiLU's one).
__device__ __forceinline__ Fp8Two fp8_rounded_product(Fp8Two a, Fp8Two b)
{
    uint32_t sm;
    asm("mov.u32 %0, %%smid;" : "=r"(sm));
    return fp8_fma(a, b, Fp8Two(__uint_as_float(0x80000000u | sm >> 20)));
}

// 1 / x for x >= 1: a Newton step with fused multiply-adds (Markstein, 1990) from the hardware's estimate, which leaves the number nearest to it where that is normal.
__device__ __forceinline__ Fp8Two fp8_reciprocal(Fp8Two x)
{
    const float2 f = x.both();
    float2 r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r.x) : "f"(f.x));
    asm("rcp.approx.f32 %0, %1;" : "=f"(r.y) : "f"(f.y));
    const Fp8Two near(r.x, r.y);
    const float2 better = fp8_fma(near, fp8_fma(x * Fp8Two(-1.0f), near, Fp8Two(1.0f)), near).both();
    return {f.x > 0x1p126f ? r.x : better.x, f.y > 0x1p126f ? r.y : better.y};  // no step from infinity's 0
}

// sigma, and the derivative of g sigma: sigma + g sigma (1 - sigma) p'.  What is made of these is quantized to three bits, where an error of 2^-22 turns one number of 2^18 into its neighbour, a
// sixteenth away; so, unlike above, every step is rounded to nearest, in the order in which the formula stands, as elementary operations in 32 bits do it.
template <bool GELU>
__device__ __forceinline__ void fp8_gate_and_slope(Fp8Two g, Fp8Two &sigma, Fp8Two &derivative)
{
    const Fp8Two one(1.0f), square = g * g;
    const float2 p = (GELU ? Fp8Two(kGeluA) * (g + fp8_rounded_product(Fp8Two(kGeluB), square * g)) : g).both();
    sigma = fp8_reciprocal(one + Fp8Two(expf(-p.x), expf(-p.y)));
    const Fp8Two a = g * sigma, b = fp8_fma(sigma, Fp8Two(-1.0f), one);
    Fp8Two rest;
    if (GELU) {  // where sigma has become 0 or 1 rest is 0, whatever p' is
        rest = a * b;
        const float2 r = rest.both(), slope = (rest * (Fp8Two(kGeluA) * (one + fp8_rounded_product(Fp8Two(kGeluB3), square)))).both();
        rest = {r.x == 0.0f ? r.x : slope.x, r.y == 0.0f ? r.y : slope.y};
    } else {
        const float2 l = a.both(), r = b.both();
        rest = {__fmul_rn(l.x, r.x), __fmul_rn(l.y, r.y)};
    }
    derivative = sigma + rest;
}

}  // namespace tuna
