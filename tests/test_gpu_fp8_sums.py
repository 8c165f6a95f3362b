"""How exact the long sums of the 8-bit products are.

The tensor cores add to an accumulator in fp32 and cut off what is below its last bit, so every addition leaves a sum nearer to zero, and a long sum is off by more than its
length has roundings.  The kernels therefore add up parts of at most 1024 addends in registers, to nearest.  Then a sum's error is that of its parts - errors of one sign add up as the parts
themselves do at worst, so relative to the sum's size it is a part's - and of the additions of P parts, each off by at most half a step, 2^-24, of what has been added up, which for addends of
any sign together are sqrt(P) 2^-24 of the sum's size.  What a part is off by is measured here with sums of one part, of the same kind of numbers."""

import math
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import tuna_b200
from oracle import fp8_oracle as fo
from tests.fp8_util import check, gated, gated_gradient, numpy64, quantized_range, rounded, sums
from tests.mx_util import HALF_STEP
from tuna_b200 import _lib

pytestmark = pytest.mark.gpu
PART = 1024
HALF_STEP32 = 2.0 ** -24


def finish():
    torch.cuda.synchronize()
    assert _lib.load().tuna_check_device_status(torch.cuda.current_stream().cuda_stream) == 0


def numbers(q, s, blocks):
    o = torch.empty(q.shape, device="cuda")
    tuna_b200.fp8_dequant(q, s, o, *q.shape, blocks)
    return o.double()


def error(got, want):
    return float((got.double() - want).norm() / want.norm())


def summed(form, length, tokens, seed):
    """(a result in 32 bits whose sums have `length` addends, what it is in 64 bits)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    other = 512
    new = lambda *shape: torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    if form == "product":
        x, w = tuna_b200.fp8_quantize(new(tokens, length)), tuna_b200.fp8_quantize(new(other, length), "square")
        o = torch.empty(tokens, other, device="cuda")
        tuna_b200.fp8_matmul(*x, *w, o, other, tokens, length)
        return o, numbers(*x, "row") @ numbers(*w, "square").T
    if form == "gated":  # z, so to speak: the gate is open everywhere, so h is the other projection
        x, w = new(tokens, length), new(2 * other, length)
        x[:, 0], w[:other] = 448.0, 0.0
        w[:other, 0] = 448.0
        x, w = tuna_b200.fp8_quantize(x), tuna_b200.fp8_quantize(w, "square")
        h = torch.empty(tokens, other, device="cuda")
        tuna_b200.fp8_gated(*x, *w, h, other, tokens, length)
        z = numbers(*x, "row") @ numbers(*w, "square").T
        assert (z[:, :other] == 448.0 ** 2).all()
        return h, z[:, :other] * z[:, other:]
    if form == "dx":
        dy, w = new(tokens, length), tuna_b200.fp8_quantize(new(length, other), "square")
        dx = torch.empty(tokens, other, device="cuda")
        tuna_b200.fp8_matmul_backward(dy, None, None, *w, dx, None, length, tokens, other)
        return dx, numbers(*tuna_b200.fp8_quantize(dy), "row") @ numbers(*w, "square")
    dy, x = new(length, tokens * 16), new(length, other)
    dw = torch.empty(tokens * 16, other, device="cuda")
    tuna_b200.fp8_matmul_backward(dy, x, None, None, None, None, dw, tokens * 16, length, other)
    return dw, numbers(*tuna_b200.fp8_quantize(dy, "column"), "column").T @ numbers(*tuna_b200.fp8_quantize(x, "column"), "column")


@pytest.mark.parametrize("length", [2048, 2176, 4096, 8192, 16384, 16400, 28672])
@pytest.mark.parametrize("tokens", [1, 16, 40, 200])
@pytest.mark.parametrize("form", ["product", "gated", "dx", "dw"])
def test_a_long_sum_is_as_exact_as_its_parts(form, tokens, length):
    of_a_part = error(*summed(form, PART, max(tokens, 16), 1))  # enough numbers for a mean
    got, want = summed(form, length, tokens, 2)
    finish()
    # one output in 512 x tokens, the mean of as many squares: 1 / sqrt(512) is a standard deviation's, and three of them are 1.15
    assert error(got, want) <= 1.15 * (of_a_part + math.sqrt(math.ceil(length / PART)) * HALF_STEP32)


@pytest.mark.parametrize("tokens", [3, 40, 200])
def test_sums_of_one_sign(tokens):
    """Every addition cuts off something, and all of it in one direction."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    off = {}
    for length in (PART, 28672):
        x, w = (torch.rand(rows, length, generator=gen, device="cuda", dtype=torch.float16) for rows in (tokens, 400))
        x, w = tuna_b200.fp8_quantize(x), tuna_b200.fp8_quantize(w, "square")
        o = torch.empty(tokens, 400, device="cuda")
        tuna_b200.fp8_matmul(*x, *w, o, 400, tokens, length)
        off[length] = error(o, numbers(*x, "row") @ numbers(*w, "square").T)
    finish()
    # what has been added up grows evenly: P additions are off by half a step of half the sum in the mean, all in one direction at worst
    assert off[28672] <= off[PART] + 28 / 2 * HALF_STEP32


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("tokens,k", [(16, 8192), (16, 16384), (200, 4096), (200, 8192), (200, 16384)])
def test_projections_that_are_kept_are_rounded_as_sums_in_32_bits_are(tokens, k, dtype):
    """z differs from the rounding of the exact sum where that lies within the sum's error of the border of two numbers: a fraction of 2 |error| over a step of them."""
    gen = torch.Generator(device="cuda").manual_seed(k)
    f = 512
    x = torch.randn(tokens, k, generator=gen, device="cuda").to(dtype)
    q, s = tuna_b200.fp8_quantize(torch.randn(2 * f, k, generator=gen, device="cuda") * k ** -0.5, "square")
    h, z = torch.empty(tokens, f, device="cuda", dtype=dtype), torch.empty(tokens, 2 * f, device="cuda", dtype=dtype)
    tuna_b200.fp8_gated(x, None, q, s, h, f, tokens, k, z=z)
    finish()
    want = numbers(*tuna_b200.fp8_quantize(x), "row") @ numbers(q, s, "square").T
    off = 1.15 * (error(*summed("product", PART, 40, 1)) + math.sqrt(math.ceil(k / PART)) * HALF_STEP32) * float(want.square().mean().sqrt())
    step = torch.ldexp(torch.ones_like(want), torch.frexp(want).exponent) * HALF_STEP[dtype][0]
    expected = float((2 * off / step).clamp(max=1).sum())
    assert int((z != want.to(dtype)).sum()) <= expected + 4 * math.sqrt(expected) + 4


@pytest.mark.parametrize("kind", ["silu", "gelu"])
@pytest.mark.parametrize("n,f,k", [(9, 400, 8192), (150, 272, 8192), (300, 144, 4112), (2100, 128, 1040)])
def test_a_gated_step_of_long_sums(n, f, k, kind):
    """Forward pass and gradients end to end: z and h against 64 bits, and the gradients for the z that was kept."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    q, s = tuna_b200.fp8_quantize(torch.randn(2 * f, k, generator=gen, device="cuda") * k ** -0.5, "square")
    x, dh = torch.randn(n, k, generator=gen, device="cuda").half(), torch.randn(n, f, generator=gen, device="cuda").half()
    h, z = torch.empty(n, f, device="cuda", dtype=torch.float16), torch.empty(n, 2 * f, device="cuda", dtype=torch.float16)
    dx, dw = torch.empty(n, k, device="cuda"), torch.empty(2 * f, k, device="cuda")
    tuna_b200.fp8_gated(x, None, q, s, h, f, n, k, kind, z=z)
    tuna_b200.fp8_gated_backward(dh, z, x, None, q, s, dx, dw, f, n, k, kind)
    finish()
    w = numpy64(numbers(q, s, "square"))
    ref_z, z_off, ref_h, h_off = gated(fo.numbers(numpy64(x), "row"), w, kind)
    check(z, ref_z, rounded(ref_z, z_off, z.dtype))
    check(h, ref_h, rounded(ref_h, h_off, h.dtype))
    dy, off = gated_gradient(numpy64(dh), numpy64(z), kind)
    a, a_off = quantized_range(dy, off, "row")
    ref, sum_off = sums(a, w, a_off)
    check(dx, ref, rounded(ref, sum_off, dx.dtype))
    b, b_off = quantized_range(dy, off, "column")
    ref, sum_off = sums(b.T, fo.numbers(numpy64(x), "column"), b_off.T)
    check(dw, ref, rounded(ref, sum_off, dw.dtype))
    assert np.isfinite(ref).all()


FIRST_CALL_CAPTURED = """
import torch, tuna_b200 as t
f, n, k = 512, 200, 8192
x, dh = (torch.randn(n, c, device="cuda", dtype=torch.bfloat16) for c in (k, f))
w = torch.randn(2 * f, k, device="cuda") * k ** -0.5
h, z = (torch.empty(n, c, device="cuda", dtype=torch.bfloat16) for c in (f, 2 * f))
o, dx, dw = (torch.empty(s, device="cuda") for s in ((n, 2 * f), (n, k), (2 * f, k)))
def step():
    q, s = t.fp8_quantize(w, "square")
    t.fp8_gated(x, None, q, s, h, f, n, k, z=z)
    t.fp8_matmul(x, None, q, s, o, 2 * f, n, k)
    t.fp8_gated_backward(dh, z, x, None, q, s, dx, dw, f, n, k)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    step()
g.replay()
torch.cuda.synchronize()
first = [v.clone() for v in (h, z, o, dx, dw)]
step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) and a.isfinite().all() for a, b in zip(first, (h, z, o, dx, dw)))
print("captured")
"""


def test_first_calls_of_long_sums_can_be_captured():
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parents[1], env=dict(os.environ))
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr
