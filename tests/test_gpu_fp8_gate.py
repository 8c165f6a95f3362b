"""The activations of the 8-bit gated block, step by step: results in 32 bits, results in 16 bits far down, and the reciprocal that the gradients divide by."""

import re
from pathlib import Path

import numpy as np
import pytest
import torch

import tuna_b200
from tests.fp8_util import numpy64
from tuna_b200 import _lib, build

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -23
KINDS = ["silu", "gelu"]
F = 128


def gates(n, lowest):
    """A block whose gates are exact, products of two e4m3 numbers, and whose other projection is one: (x, w, gates [n, F])."""
    a = torch.linspace(-1, 0.35, F) * 448
    b = torch.linspace(1 / 16, 1, n) * -lowest / 448
    x, w = torch.zeros(n, 128), torch.zeros(2 * F, 128)
    x[:, 0], x[:, 1] = b, 1 / 16
    w[:F, 0], w[F:, 1] = a, 16
    x, w = tuna_b200.fp8_quantize(x.cuda()), tuna_b200.fp8_quantize(w.cuda(), "square")
    as_numbers = []
    for (q, s), blocks in ((x, "row"), (w, "square")):
        o = torch.empty(q.shape, device="cuda")
        tuna_b200.fp8_dequant(q, s, o, *q.shape, blocks)
        as_numbers.append(numpy64(o))
    z = as_numbers[0] @ as_numbers[1].T
    assert (z[:, F:] == 1).all() and z[:, :F].min() < 0.95 * lowest
    return x, w, z[:, :F]


def argument(g, kind):
    return g if kind == "silu" else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)


def block(x, w, n, dtype, kind):
    h = torch.full((n, F), float("nan"), device="cuda", dtype=dtype)
    tuna_b200.fp8_gated(*x, *w, h, F, n, 128, kind)
    torch.cuda.synchronize()
    assert _lib.load().tuna_check_device_status(torch.cuda.current_stream().cuda_stream) == 0
    return numpy64(h)


def exact(g, kind):
    """g sigma(p(g)), also where sigma is far below one (the oracle's form of GELU, 1 + tanh, loses it there)."""
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-argument(g, kind)))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [3, 16, 60, 300])
def test_results_in_32_bits_are_those_of_elementary_operations(n, kind):
    """The exponential is off by two steps at most, the sum, the quotient and the product by half a step each: 3.5, and of GELU the argument by six roundings, which the exponential
    multiplies by it.  Where 1 / (1 + exp) is below fp32's normal numbers it is rounded to a multiple of 2^-149, and where the exponential overflows, it is 0."""
    x, w, g = gates(n, -100.0 if kind == "silu" else -9.0)
    p = np.abs(argument(g, kind))
    tol = (4 + (3 * p if kind == "gelu" else 0)) * STEP * np.abs(exact(g, kind)) + np.abs(g) * np.where(argument(g, kind) < -88.7, 2.0 ** -127, 2.0 ** -149)
    assert (np.abs(block(x, w, n, torch.float32, kind) - exact(g, kind)) <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [3, 16, 60, 300])
def test_results_in_16_bits_are_right_to_the_last_that_there_are(n, kind, dtype):
    """The hardware's exponential is off by 2 + 1.2 |p| steps, the rest by two; GELU's argument as above; then one rounding.  Below 2^-126 the logistic function is 0."""
    x, w, g = gates(n, -100.0 if kind == "silu" else -9.0)
    want, p = exact(g, kind), np.abs(argument(g, kind))
    off = (4 + 1.2 * p + (3 * p if kind == "gelu" else 0)) * STEP * np.abs(want) + np.abs(g) * np.where(argument(g, kind) < -87.3, 2.0 ** -126, 2.0 ** -149)
    half, least = (2.0 ** -11, 2.0 ** -25) if dtype == torch.float16 else (2.0 ** -8, 2.0 ** -134)  # half a step; half of the smallest number
    got = block(x, w, n, dtype, kind)
    assert (np.abs(got - want) <= off + half * (np.abs(want) + off) + least).all()
    if dtype == torch.bfloat16:
        assert (got != 0)[(argument(g, kind) > -87) & (g != 0)].all()


PROGRAM = """
typedef unsigned int uint32_t;
typedef unsigned long long uint64_t;
%s
// out[0]: how many reciprocals of the numbers 2^e (1 + m 2^-23) are not the nearest, out[1]: the bits of one of them
extern "C" __global__ void reciprocals(int e, unsigned int *out)
{
    const unsigned int m = blockIdx.x * blockDim.x + threadIdx.x;
    const float x = __uint_as_float((unsigned int)(e + 127) << 23 | m), y = __uint_as_float((unsigned int)(e + 127) << 23 | (m * 2654435761u & 0x7fffffu));
    const float2 r = tuna::fp8_reciprocal(tuna::Fp8Two(x, y)).both();
    if (r.x != 1.0f / x || r.y != 1.0f / y) {
        atomicAdd(out, 1u);
        out[1] = __float_as_uint(r.x != 1.0f / x ? x : y);
    }
}
"""


@pytest.fixture(scope="module")
def reciprocals():
    text = re.sub(r"^\s*#pragma once.*$", "", (Path(build.CSRC) / "fp8_gate.cuh").read_text(), flags=re.M)
    assert "#include" not in text
    return torch.cuda._compile_kernel(PROGRAM % text, "reciprocals")


@pytest.mark.parametrize("e", [0, 1, 2, 24, 63, 100, 124, 125])
def test_the_reciprocal_is_the_nearest_number(reciprocals, e):
    """Of every significand: the quotient that torch's division gives."""
    out = torch.zeros(2, dtype=torch.int32, device="cuda")
    reciprocals(grid=(1 << 15, 1, 1), block=(256, 1, 1), args=[e, out])
    count, bits = out.tolist()
    assert count == 0, f"{count} of 2^24, among them {bits:#x}"


def test_the_reciprocals_ends(reciprocals):
    """From 2^126 on the nearest number is not normal: the estimate stands."""
    source = PROGRAM.replace("extern", """extern "C" __global__ void at(const float *x, float *r, int n) { for (int i = 0; i < n; ++i) r[i] = tuna::fp8_reciprocal(tuna::Fp8Two(x[i])).both().x; }
extern""", 1)
    text = re.sub(r"^\s*#pragma once.*$", "", (Path(build.CSRC) / "fp8_gate.cuh").read_text(), flags=re.M)
    run = torch.cuda._compile_kernel(source % text, "at")
    x = torch.tensor([1.0, 2.0 ** 126, 2.0 ** 126 * 1.5, 2.0 ** 127 * 1.99, float("inf"), 2 - 2.0 ** -23], device="cuda")
    r = torch.empty_like(x)
    run(grid=(1, 1, 1), block=(1, 1, 1), args=[x, r, x.numel()])
    want = 1 / x.double()
    assert ((r.double() - want).abs() <= 2.0 ** -24 * want + 2.0 ** -148).all()


ROUNDED = """
typedef unsigned int uint32_t;
typedef unsigned long long uint64_t;
%s
// out: how many of c + a b are not rounded twice, and how many of them a fused step would give
extern "C" __global__ void rounded(const float *a, const float *b, const float *c, double minus_zero, int *out)
{
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    const tuna::Fp8Two sum = tuna::Fp8Two(c[i]) + tuna::fp8_rounded_product(tuna::Fp8Two(a[i]), tuna::Fp8Two(b[i]), (float)minus_zero);
    if (sum.both().x != __fadd_rn(c[i], __fmul_rn(a[i], b[i]))) atomicAdd(out, 1);
    if (__fmaf_rn(a[i], b[i], c[i]) != __fadd_rn(c[i], __fmul_rn(a[i], b[i]))) atomicAdd(out + 1, 1);
}
"""


def test_a_product_that_is_added_is_rounded_first():
    text = re.sub(r"^\s*#pragma once.*$", "", (Path(build.CSRC) / "fp8_gate.cuh").read_text(), flags=re.M)
    run = torch.cuda._compile_kernel(ROUNDED % text, "rounded")
    gen = torch.Generator(device="cuda").manual_seed(0)
    a, b, c = (torch.randn(1 << 20, generator=gen, device="cuda") for _ in range(3))
    out = torch.zeros(2, dtype=torch.int32, device="cuda")
    run(grid=(1 << 12, 1, 1), block=(256, 1, 1), args=[a, b, c, -0.0, out])
    wrong, fused = out.tolist()
    assert wrong == 0 and fused > 1 << 16  # these numbers tell one from the other
