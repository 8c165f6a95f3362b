"""Shared by the tests of the microscaled operators: random matrices of every kind, and how far a product may be off."""

import numpy as np
import torch

from oracle import mx_oracle as mxo

#: half a step of rounding to nearest, relative, and the smallest subnormal's half (2^-25 of fp16, 2^-134 of bf16, 2^-150 of fp32)
HALF_STEP = {torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float32: (2.0 ** -24, 2.0 ** -150)}


def random_packed(rows, k, seed, spread=3):
    """A matrix of random codes, all sixteen of them, and scales 2^-spread .. 2^spread: packed, and its numbers in 64 bits."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (rows, k), dtype=np.uint8)
    scales = rng.integers(127 - spread, 128 + spread, (rows, k // 32), dtype=np.uint8)
    return mxo.pack(codes, scales), mxo.decode(codes, scales)


def allowed(x, w, dtype):
    """(exact product, what a result may be off): every product of two numbers is exact in fp32 (six significant bits).  The k of
    them are added in fp32 in some order, each addition off by at most a step, 2^-23, of what has been added up so far, which the
    sum of magnitudes bounds; then one rounding to `dtype`."""
    ref = x @ w.T
    magnitude = np.abs(x) @ np.abs(w).T
    summed = x.shape[1] * 2.0 ** -23 * magnitude
    rel, tiny = HALF_STEP[dtype]
    return ref, summed + rel * (np.abs(ref) + summed) + tiny


def check_product(o, x, w):
    """`o` (a tensor) against x [n, k] times w [m, k] transposed in 64 bits."""
    ref, tol = allowed(x, w, o.dtype)
    out = o.double().cpu().numpy()
    assert np.array_equal(np.isnan(out), np.isnan(ref))
    off = np.abs(out - ref)
    bad = ~(off <= tol) & ~np.isnan(ref)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, first at {np.argwhere(bad)[0]}: {out[bad][0]} is not {ref[bad][0]} +- {tol[bad][0]}"
