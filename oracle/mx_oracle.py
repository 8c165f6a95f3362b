"""CPU oracle for the microscaled 4-bit (OCP MXFP4) operators: numpy in 64 bits, written from the format's definition.

TEST INFRASTRUCTURE ONLY, like the rest of this folder.  A number is an e2m1 code (bit 3 the sign, bits 2-1 the exponent, bit 0
the mantissa) times 2^(b - 127), b the scale byte of its block of 32 columns (255: NaN).
"""

from __future__ import annotations

import numpy as np

#: The eight magnitudes, from the fields: exponent 0 is subnormal (mantissa / 2), else 2^(exponent - 1) (1 + mantissa / 2).
MAGNITUDES = np.array([m / 2 if e == 0 else 2.0 ** (e - 1) * (1 + m / 2) for e in range(4) for m in range(2)])


def encode(v: np.ndarray) -> np.ndarray:
    """Codes nearest to `v`, ties to the even code, saturating at 6."""
    a = np.abs(v)[..., None]
    distance = np.abs(a - MAGNITUDES)
    best = distance.min(-1, keepdims=True)
    near = distance == best  # two of them at a tie
    even = np.arange(8) % 2 == 0
    code = np.where((near & even).any(-1) & (near.sum(-1) > 1), np.argmax(near & even, -1), np.argmax(near, -1))
    return (code | (np.signbit(v).astype(np.int64) << 3)).astype(np.uint8)


def quantize(x: np.ndarray):
    """[rows, k] -> row-major codes [rows, k] (one a byte) and scale bytes [rows, k / 32]."""
    rows, k = x.shape
    v = x.astype(np.float64).reshape(rows, k // 32, 32)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0.0, v)
    largest = np.abs(v).max(-1)
    _, exponent = np.frexp(largest)  # largest = f 2^exponent with f in [0.5, 1)
    e = np.where(largest > 0, np.maximum(exponent - 1 - 2, -127), -127)
    codes = encode(v / np.ldexp(1.0, e)[..., None])
    return codes.reshape(rows, k), np.where(bad, 255, e + 127).astype(np.uint8)


def decode(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    v = MAGNITUDES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return v * np.repeat(s, 32, axis=-1)


def pack(codes: np.ndarray, scales: np.ndarray):
    """The package's layout: q [ceil(k/256), rows, 128], s [ceil(k/128), rows, 4], zeros behind column k."""
    rows, k = codes.shape
    q = np.zeros((-(-k // 256), rows, 128), dtype=np.uint8)
    s = np.zeros((-(-k // 128), rows, 4), dtype=np.uint8)
    for c in range(k):
        q[c // 256, :, c % 256 // 2] |= codes[:, c] << (4 * (c % 2))
    for b in range(k // 32):
        s[b // 4, :, b % 4] = scales[:, b]
    return q, s


def unpack(q: np.ndarray, s: np.ndarray, k: int):
    rows = q.shape[1]
    codes = np.zeros((rows, k), dtype=np.uint8)
    scales = np.zeros((rows, k // 32), dtype=np.uint8)
    for c in range(k):
        codes[:, c] = (q[c // 256, :, c % 256 // 2] >> (4 * (c % 2))) & 15
    for b in range(k // 32):
        scales[:, b] = s[b // 4, :, b % 4]
    return codes, scales
