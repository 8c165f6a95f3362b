"""Microscaled products whose sums are exact in 24 bits in any order: a result has to be the 64-bit one, rounded once.

Numbers are multiples of 2^-2 (codes of 2^-1, scales from 2^-1 on), so products are multiples of 2^-4, and every case checks that the
magnitudes of a result's products add up to less than 2^24 of these.  No partial sum then needs more than the 24 bits of fp32,
whatever is added to what first; an accumulator of fewer bits, or a rounding between steps, shows.
"""

import numpy as np
import pytest
import torch

import tuna_b200
from tests.gpu_util import stream_ptr
from oracle import mx_oracle as mxo
from tuna_b200 import _lib

pytestmark = pytest.mark.gpu


def numbers(rows, k, seed, positive):
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 8 if positive else 16, (rows, k), dtype=np.uint8)
    scales = rng.integers(126, 129, (rows, k // 32), dtype=np.uint8)
    return codes, scales


def matrix(rows, k, seed, positive, distinct=96):
    """Packed codes on the GPU and numbers in 64 bits of `rows` rows, of which so many differ."""
    codes, scales = numbers(min(rows, distinct), k, seed, positive)
    turn = np.arange(rows) % len(codes)
    q, s = (torch.from_numpy(np.ascontiguousarray(a[:, turn])).cuda() for a in mxo.pack(codes, scales))
    return (q, s), mxo.decode(codes, scales), turn


def same(o, x, w, turn_x, turn_w):
    assert (np.abs(x) @ np.abs(w).T).max() * 16 < 2 ** 24
    exact = torch.from_numpy((x @ w.T)[turn_x][:, turn_w])
    torch.cuda.synchronize()
    assert _lib.load().tuna_check_device_status(stream_ptr()) == 0
    assert torch.equal(o.cpu(), exact.to(o.dtype))  # 64 bits -> o's type: one rounding


# up to 16 tokens: four, two chunks side by side, one; more: tiles of up to 64, 128, 160 to 192 and 256 tokens on pairs of CTAs
FORMS = [(264, 1), (264, 3), (264, 16), (7000, 16), (9600, 5), (9600, 16), (520, 40), (520, 100), (2048, 170), (4096, 300), (264, 1000)]


@pytest.mark.parametrize("positive", [False, True], ids=["signed", "positive"])
@pytest.mark.parametrize("k", [4096, 14336, 28672])
@pytest.mark.parametrize("m,n", FORMS)
def test_sums_of_codes(m, n, k, positive):
    w, wn, tw = matrix(m, k, 1, positive)
    x, xn, tx = matrix(n, k, 2, positive)
    for dtype in (torch.float32, torch.bfloat16):
        o = torch.full((n, m), float("nan"), device="cuda", dtype=dtype)
        tuna_b200.mx_matmul(*x, *w, o, m, n, k)
        same(o, xn, wn, tx, tw)


@pytest.mark.parametrize("k", [4096, 14336, 28672])
@pytest.mark.parametrize("m,n", [(264, 1), (264, 2), (9600, 1), (264, 16), (520, 100)])
def test_sums_of_tokens_in_16_bits(m, n, k):
    """Numbers that bf16 holds, each block with a 6, so that quantizing gives them back."""
    w, wn, tw = matrix(m, k, 3, False)
    codes, scales = numbers(min(n, 96), k, 4, False)
    codes[:, ::32] = 7
    xn = mxo.decode(codes, scales)
    tx = np.arange(n) % len(codes)
    x = torch.from_numpy(xn[tx]).to(torch.bfloat16).cuda()
    o = torch.full((n, m), float("nan"), device="cuda")
    tuna_b200.mx_matmul(x, None, *w, o, m, n, k)
    same(o, xn, wn, tx, tw)


@pytest.mark.parametrize("k", [4096, 14336, 28672])
@pytest.mark.parametrize("counts", [[3, 0, 20], [70, 90, 1], [300, 5, 200]], ids=str)
def test_sums_of_experts(counts, k):
    m, n = 264, sum(counts)
    mats = [matrix(m, k, 10 + e, False) for e in range(len(counts))]
    q, s = (torch.stack([p[0][i] for p in mats]) for i in (0, 1))
    x, xn, tx = matrix(n, k, 5, False)
    ends = np.cumsum([0] + counts)
    o = torch.full((n, m), float("nan"), device="cuda")
    tuna_b200.mx_matmul_grouped(*x, q, s, torch.from_numpy(ends.astype(np.int32)).cuda(), o, m, n, k)
    for e, (_, wn, tw) in enumerate(mats):
        if counts[e]:
            same(o[ends[e]:ends[e + 1]], xn, wn, tx[ends[e]:ends[e + 1]], tw)


# ------------------------------------------------------------------ scales at both ends

EXTREMES = [0, 1, 2, 27, 126, 127, 128, 227, 252, 253, 254]


def opposite(rows, k, seed, bytes_of_blocks):
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 16, (rows, k), dtype=np.uint8)
    return codes, np.broadcast_to(bytes_of_blocks, (rows, k // 32)).astype(np.uint8)


def end_scales(k, seed):
    """A byte for every block of the tokens and the one of the weights that makes the scales' product 1, 2 or 1/2."""
    rng = np.random.default_rng(seed)
    a = rng.permutation(np.resize(EXTREMES, k // 32))
    b = np.clip(254 - a + rng.integers(-1, 2, k // 32), 0, 254)
    return a, b


@pytest.mark.parametrize("m,n", [(264, 1), (264, 16), (9600, 16), (520, 40), (520, 130), (1000, 300)])
def test_scales_at_both_ends(m, n):
    """2^-127 x 2^127 and everything between: products of scales near 1, so sums are exact as above (products are multiples of 2^-3)."""
    k = 1056
    a, b = end_scales(k, m)
    for x_bytes, w_bytes in ((a, b), (b, a)):
        xc, wc = opposite(min(n, 96), k, 1, x_bytes), opposite(min(m, 96), k, 2, w_bytes)
        tx, tw = np.arange(n) % len(xc[0]), np.arange(m) % len(wc[0])
        xq, xs, q, s = (torch.from_numpy(np.ascontiguousarray(t[:, turn])).cuda() for p, turn in ((mxo.pack(*xc), tx), (mxo.pack(*wc), tw)) for t in p)
        o = torch.full((n, m), float("nan"), device="cuda")
        tuna_b200.mx_matmul(xq, xs, q, s, o, m, n, k)
        same(o, mxo.decode(*xc), mxo.decode(*wc), tx, tw)
        two = torch.full((n, m), float("nan"), device="cuda")
        off = torch.tensor([0, n // 2, n], dtype=torch.int32, device="cuda")
        tuna_b200.mx_matmul_grouped(xq, xs, torch.stack([q, q]), torch.stack([s, s]), off, two, m, n, k)
        torch.cuda.synchronize()
        assert torch.equal(o, two)


@pytest.mark.parametrize("n", [1, 2, 16, 40])
def test_tokens_in_16_bits_with_scales_at_both_ends(n):
    """Tokens of up to 6 x 2^-126 in one block and 6 x 2^125 in another, whose scales the call finds, against weights with the opposite scales."""
    m, k = 264, 1056
    a = np.random.default_rng(n).permutation(np.resize([1, 2, 27, 127, 227, 251, 252], k // 32))
    codes, scales = opposite(n, k, 3, a)
    codes[:, ::32] = 7
    xn = mxo.decode(codes, scales)
    x = torch.from_numpy(xn).to(torch.bfloat16).cuda()
    wc = opposite(m, k, 4, 254 - a)
    q, s = (torch.from_numpy(t).cuda() for t in mxo.pack(*wc))
    o = torch.full((n, m), float("nan"), device="cuda")
    tuna_b200.mx_matmul(x, None, q, s, o, m, n, k)
    same(o, xn, mxo.decode(*wc), np.arange(n), np.arange(m))
