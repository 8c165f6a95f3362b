"""The activations of the 8-bit gated block, step by step: results in 32 bits, and results in 16 bits far down."""

import numpy as np
import pytest
import torch

import tuna_b200
from tests.fp8_util import numpy64
from tuna_b200 import _lib

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

