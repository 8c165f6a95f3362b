"""CPU oracle for the 8-bit block-scaled operators: numpy in 64 bits, written from the format's definition.

TEST INFRASTRUCTURE ONLY, like the rest of this folder.  A number is an e4m3 code (bit 7 the sign, bits 6-3 the exponent, bits 2-0
the mantissa; 0x7f and 0xff are NaN) times 2^(b - 127), b the scale byte of its block (255: NaN).  Blocks are 128 columns of a row, 128 rows
of a column, or square.
"""

from __future__ import annotations

import numpy as np

#: The magnitudes of codes 0 .. 126, from the fields: exponent 0 is subnormal (mantissa 2^-9), else 2^(exponent - 7) (1 + mantissa / 8).
MAGNITUDES = np.array([m * 2.0 ** -9 if e == 0 else 2.0 ** (e - 7) * (1 + m / 8) for e in range(16) for m in range(8)][:127])
SHAPES = {"row": (1, 128), "column": (128, 1), "square": (128, 128)}


def encode(v: np.ndarray) -> np.ndarray:
    """Codes nearest to `v`, ties to the even code, saturating at 448."""
    a = np.minimum(np.abs(v), 448.0)
    up = np.clip(np.searchsorted(MAGNITUDES, a), 0, 126)  # the first magnitude not below
    down = np.maximum(up - 1, 0)
    above, below = MAGNITUDES[up] - a, a - MAGNITUDES[down]
    code = np.where((above < below) | ((above == below) & (up % 2 == 0)), up, down)
    return (code | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def spread(s: np.ndarray, blocks: str, rows: int, k: int) -> np.ndarray:
    """One value per block -> one per element."""
    r, c = SHAPES[blocks]
    return np.repeat(np.repeat(s, r, 0), c, 1)[:rows, :k]


def largest(a: np.ndarray, blocks: str) -> np.ndarray:
    """Of every block's magnitudes `a`."""
    r, c = SHAPES[blocks]
    rows, k = a.shape
    p = np.zeros((-(-rows // r) * r, -(-k // c) * c))
    p[:rows, :k] = a
    return p.reshape(p.shape[0] // r, r, p.shape[1] // c, c).max((1, 3))


def scale_of(a: np.ndarray) -> np.ndarray:
    """The exponent of the smallest power of two over which `a` is not above 448, at least -127."""
    _, e = np.frexp(a / 448.0)  # a / 448 = f 2^e with f in [0.5, 1): 448 2^(e - 1) is enough where f is 0.5
    e = np.where(a <= np.ldexp(448.0, e - 1), e - 1, e)
    return np.where(a > 0, np.maximum(e, -127), -127)


def quantize(x: np.ndarray, blocks: str):
    """[rows, k] -> codes [rows, k] and scale bytes, one per block [blocks of rows, blocks of columns]."""
    v = x.astype(np.float64)
    bad = largest((~np.isfinite(v)).astype(float), blocks) > 0
    v = np.where(np.isfinite(v), v, 0.0)
    e = scale_of(largest(np.abs(v), blocks))
    codes = encode(v / np.ldexp(1.0, spread(e, blocks, *x.shape)))
    codes = np.where(spread(bad, blocks, *x.shape), 0, codes).astype(np.uint8)
    return codes, np.where(bad, 255, e + 127).astype(np.uint8)


def decode(codes: np.ndarray, scales: np.ndarray, blocks: str) -> np.ndarray:
    v = np.append(MAGNITUDES, np.nan)[codes & 127] * np.where(codes & 128, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return v * spread(s, blocks, *codes.shape)


def numbers(x: np.ndarray, blocks: str) -> np.ndarray:
    return decode(*quantize(x, blocks), blocks)


def pack(scales: np.ndarray, blocks: str) -> np.ndarray:
    """The package's layout of one byte per block: words of four blocks, zeros behind the last."""
    if blocks == "square":
        return scales
    s = scales.T if blocks == "row" else scales  # [blocks along what is summed over, across]
    out = np.zeros((-(-s.shape[0] // 4), s.shape[1], 4), dtype=np.uint8)
    for b in range(s.shape[0]):
        out[b // 4, :, b % 4] = s[b]
    return out


def activation(g: np.ndarray, kind: str):
    """(value, derivative) of SiLU, or of GELU in its tanh form."""
    if kind == "silu":
        with np.errstate(over="ignore"):
            s = 1 / (1 + np.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    c = np.sqrt(2 / np.pi)
    t = np.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
