// The activations of a gated block on the device, and their derivatives.  It includes nothing (the integer types are there already): a test compiles it by itself.
#pragma once

namespace tuna {

// The activation is g * sigma(p(g)), sigma the logistic function: p = g (SiLU) or 2 sqrt(2 / pi) (g + 0.044715 g^3) (GELU in its tanh form, as
// (1 + tanh(y)) / 2 = sigma(2 y)).
constexpr float kGeluA = 1.5957691216057308f, kGeluB = 0.044715f, kGeluB3 = 0.134145f;  // the last: three times the one before
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
// the sum with a -0 that the compiler does not know for one: an argument of the launch (gradients of 1360 features and 333 tokens 22.0 us; 22.9 with two single products, which it leaves apart
// and which are as fast for SiLU's one).
__device__ __forceinline__ Fp8Two fp8_rounded_product(Fp8Two a, Fp8Two b, float minus_zero) { return fp8_fma(a, b, Fp8Two(minus_zero)); }

// 1 / x for x >= 1, the number nearest to it where that is normal: a Newton step with fused multiply-adds (Markstein, 1990) from the hardware's estimate.  The theorem leaves out divisors whose
// significand is all ones, for which it depends on the estimate; compared with the quotient for every significand, they are right as well.
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

// sigma(p(g)).  EXACT, for results in 32 bits: the exponential to two steps, everything else rounded to nearest.  Otherwise by the hardware's exponential and a fast quotient, which are off by up to
// 4 + 1.2 |p| steps of 2^-23, a fiftieth of half a step of fp16 where that has a result at all (p > -18) and less of bf16's, and 0 where sigma is below 2^-126 (a reciprocal that has those too: gated
// 4096x2048 at 2048 tokens with z 41 -> 44 us).
template <bool GELU, bool EXACT>
__device__ __forceinline__ Fp8Two fp8_gate(float g0, float g1)
{
    const float p0 = GELU ? kGeluA * fmaf(kGeluB * g0 * g0, g0, g0) : g0, p1 = GELU ? kGeluA * fmaf(kGeluB * g1 * g1, g1, g1) : g1;
    if (EXACT) return fp8_reciprocal(Fp8Two(1.0f) + Fp8Two(expf(-p0), expf(-p1)));
    return {__fdividef(1.0f, 1.0f + __expf(-p0)), __fdividef(1.0f, 1.0f + __expf(-p1))};  // exp overflows to infinity, and the quotient is 0 then
}

// sigma, and the derivative of g sigma: sigma + g sigma (1 - sigma) p'.  What is made of these is quantized to three bits, where an error of 2^-22 turns one number of 2^18 into its neighbour, a
// sixteenth away; so, unlike above, every step is rounded to nearest, in the order in which the formula stands, as elementary operations in 32 bits do it.
template <bool GELU>
__device__ __forceinline__ void fp8_gate_and_slope(Fp8Two g, float minus_zero, Fp8Two &sigma, Fp8Two &derivative)
{
    const Fp8Two one(1.0f), square = g * g;
    const float2 p = (GELU ? Fp8Two(kGeluA) * (g + fp8_rounded_product(Fp8Two(kGeluB), square * g, minus_zero)) : g).both();
    sigma = fp8_reciprocal(one + Fp8Two(expf(-p.x), expf(-p.y)));
    const Fp8Two a = g * sigma, b = fp8_fma(sigma, Fp8Two(-1.0f), one);
    Fp8Two rest;
    if (GELU) {  // where sigma has become 0 or 1 rest is 0, whatever p' is
        rest = a * b;
        const float2 r = rest.both(), slope = (rest * (Fp8Two(kGeluA) * (one + fp8_rounded_product(Fp8Two(kGeluB3), square, minus_zero)))).both();
        rest = {r.x == 0.0f ? r.x : slope.x, r.y == 0.0f ? r.y : slope.y};
    } else {
        const float2 l = a.both(), r = b.both();
        rest = {__fmul_rn(l.x, r.x), __fmul_rn(l.y, r.y)};
    }
    derivative = sigma + rest;
}

}  // namespace tuna
