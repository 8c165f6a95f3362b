"""Shared by the tests of the 8-bit block-scaled operators: random matrices, and how far results may be off.

Where a tolerance comes from: every product of two numbers is exact in fp32 (eight significant bits).  The k of them are added in fp32 in some
order, each addition off by at most a step, 2^-23, of what has been added up so far, which the sum of magnitudes bounds; then one rounding
to the output's type, half a step.
"""

import numpy as np
import torch

from oracle import fp8_oracle as fo
from tests.mx_util import HALF_STEP

STEP32 = 2.0 ** -23
#: |derivative| of either activation is below this (1.0998 of SiLU, 1.129 of GELU), its second derivative below 1
SLOPE = 1.13


def codes_tensor(codes, device="cuda"):
    return torch.from_numpy(np.ascontiguousarray(codes)).to(device).view(torch.float8_e4m3fn)


def random_matrix(rows, k, blocks, seed, spread=3):
    """Codes and scales of every kind of number (no NaN), scales 2^-spread .. 2^spread: as the package has them on the device, and in 64 bits."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 127, (rows, k), dtype=np.uint8) | (rng.integers(0, 2, (rows, k), dtype=np.uint8) << 7)
    r, c = fo.SHAPES[blocks]
    scales = rng.integers(127 - spread, 128 + spread, (-(-rows // r), -(-k // c)), dtype=np.uint8)
    return (codes_tensor(codes), torch.from_numpy(fo.pack(scales, blocks)).cuda()), fo.decode(codes, scales, blocks)


def numpy64(t):
    return t.double().cpu().numpy()


def rounded(ref, off, dtype):
    """What a value may be off that is `ref` give or take `off` before it is rounded to `dtype`."""
    rel, tiny = HALF_STEP[dtype]
    return off + rel * (np.abs(ref) + off) + tiny


def sums(a, b, a_off=None, b_off=None):
    """(a @ b, what fp32 sums may be off), a's and b's entries being themselves off by as much as a_off and b_off say."""
    ref = a @ b
    size, off = np.abs(a), 0.0
    if a_off is not None:
        off = a_off @ np.abs(b)
        size = size + a_off
    magnitude = size @ np.abs(b)
    if b_off is not None:
        off = off + size @ b_off
        magnitude = magnitude + size @ b_off
    return ref, off + a.shape[1] * STEP32 * magnitude


#: What is not below this rounds to infinity: the largest number and half of the step above it.
OVERFLOW = {torch.float16: 65520.0, torch.bfloat16: 2.0 ** 128 * (1 - 2.0 ** -9), torch.float32: 2.0 ** 128 * (1 - 2.0 ** -25)}


def check(o, ref, tol):
    out = numpy64(o)
    assert out.shape == ref.shape
    assert np.array_equal(np.isnan(out), np.isnan(ref))
    with np.errstate(invalid="ignore"):
        over = np.isinf(out) & (np.sign(out) == np.sign(ref)) & (np.abs(ref) + tol >= OVERFLOW[o.dtype])
        bad = ~(np.abs(out - ref) <= tol) & ~np.isnan(ref) & (out != ref) & ~over
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: {out[bad][0]} is not {ref[bad][0]} +- {np.broadcast_to(tol, ref.shape)[bad][0]}"


def check_product(o, a, b):
    """`o` against a @ b."""
    ref, off = sums(a, b)
    check(o, ref, rounded(ref, off, o.dtype))


def gate_error(g, kind):
    """What fp32 makes of the activation is off by, relative: the logistic function's argument has a few roundings (five), which its exponential
    multiplies by the argument; that, the sum, the quotient and the products are off by two steps each at most."""
    p = np.abs(g) if kind == "silu" else np.abs(1.6 * (g + 0.044715 * g ** 3))
    return (12 + 5 * np.minimum(p, 200.0)) * STEP32


def gated(x, w, kind):
    """(z, what its fp32 sums may be off, h, what h may be off) for x [n, k], w [2f, k]."""
    z, off = sums(x, w.T)
    f = w.shape[0] // 2
    g, u, g_off, u_off = z[:, :f], z[:, f:], off[:, :f], off[:, f:]
    a, _ = fo.activation(g, kind)
    a_off = SLOPE * g_off + gate_error(g, kind) * np.abs(a) + 2.0 ** -126  # below fp32's range the logistic function is 0
    h = a * u
    return z, off, h, a_off * (np.abs(u) + u_off) + np.abs(a) * u_off + STEP32 * np.abs(h)


def gated_gradient(dh, z, kind):
    """([dh u activation'(g) | dh activation(g)], what fp32 may make of it is off by), all inputs exact."""
    f = dh.shape[1]
    g, u = z[:, :f], z[:, f:]
    a, d = fo.activation(g, kind)
    # the derivative is sigma + g sigma (1 - sigma) p', each term with the activation's relative error; they cancel, so it counts for each
    with np.errstate(divide="ignore", invalid="ignore"):
        sigma = np.where(g == 0, 0.5, a / g)
    terms = np.abs(sigma) + np.abs(d - sigma)
    err = gate_error(g, kind)
    dy = np.concatenate((dh * u * d, dh * a), 1)
    off = np.concatenate((np.abs(dh * u) * (2 * err * terms), np.abs(dh * a) * err), 1) + 4 * STEP32 * np.abs(dy) + 2.0 ** -126 * np.abs(np.concatenate((dh * u, dh), 1))
    return dy, off


def quantized_range(v, off, blocks):
    """Numbers that are v give or take off are quantized: (one of what they may become, how far another may be from it)."""
    small, large = fo.largest(np.maximum(np.abs(v) - off, 0), blocks), fo.largest(np.abs(v) + off, blocks)
    ends = []
    for e in (fo.scale_of(small), fo.scale_of(large)):
        s = np.ldexp(1.0, fo.spread(e, blocks, *v.shape))
        for end in (v - off, v, v + off):
            code = fo.encode(end / s)
            ends.append(np.append(fo.MAGNITUDES, np.nan)[code & 127] * np.where(code & 128, -1.0, 1.0) * s)
    ends = np.stack(ends)
    return ends[1], np.maximum(ends.max(0) - ends[1], ends[1] - ends.min(0))
