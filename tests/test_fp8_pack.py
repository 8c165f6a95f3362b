"""Checkpoints' matrices of many blocks: `fp8_pack` takes them a few million numbers at a time."""

import numpy as np
import pytest
import torch

import tuna_b200
from oracle import fp8_oracle as fo
from tuna_b200 import fp8


def checkpoint(rows, k, seed):
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 127, (rows, k), dtype=np.uint8) | (rng.integers(0, 2, (rows, k), dtype=np.uint8) << 7)
    return codes, np.exp2(rng.uniform(-12, 3, (-(-rows // 128), -(-k // 128)))).astype(np.float32)


def pack_and_check(rows, k, device):
    codes, scales = checkpoint(rows, k, rows)
    q, s = tuna_b200.fp8_pack(torch.from_numpy(codes).to(device).view(torch.float8_e4m3fn), torch.from_numpy(scales).to(device))
    assert q.shape == (rows, k) and q.is_contiguous() and s.is_contiguous()
    v = fo.decode(codes, np.full(scales.shape, 127, dtype=np.uint8), "square") * fo.spread(scales.astype(np.float64), "square", rows, k)
    want = fo.quantize(v, "square")
    assert np.array_equal(s.cpu().numpy(), want[1])
    assert np.array_equal(fo.decode(q.view(torch.uint8).cpu().numpy(), s.cpu().numpy(), "square"), fo.decode(*want, "square"))


SIZES = [(1, 16), (129, 400), (600, 16384), (128, 40000), (300, 33024)]  # one turn, several, a turn of one row of blocks


@pytest.mark.parametrize("rows,k", SIZES)
def test_matrices_of_several_turns(rows, k):
    pack_and_check(rows, k, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k", SIZES)
def test_matrices_of_several_turns_on_the_gpu(rows, k):
    pack_and_check(rows, k, "cuda")


@pytest.mark.parametrize("e,keeps", [(-127, True), (-120, True), (0, True), (119, True), (-128, False), (-140, False)])
def test_which_powers_of_two_keep_their_numbers(e, keeps):
    codes = torch.arange(127, dtype=torch.uint8)[None].repeat(2, 1)
    scales = torch.full((1, 1), 2.0 ** e, dtype=torch.float64).float()
    q, s = tuna_b200.fp8_pack(codes.view(torch.float8_e4m3fn), scales)
    numbers = fo.decode(q.view(torch.uint8).numpy(), s.numpy(), "square")
    want = fo.decode(codes.numpy(), np.full((1, 1), 127, dtype=np.uint8), "square") * 2.0 ** e
    assert np.array_equal(numbers, want) == keeps
    assert (np.abs(numbers - want) <= np.maximum(2.0 ** -4 * want, 2.0 ** -137)).all()


@pytest.mark.gpu
def test_memory_does_not_grow_with_the_matrix():
    rows, k = 8192, 8192
    codes = torch.zeros(rows, k, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.ones(rows // 128, k // 128, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    q, _ = tuna_b200.fp8_pack(codes, scales)
    used = torch.cuda.max_memory_allocated() - before
    # the result, and a turn's: a dozen numbers of 64 bits for each of its own
    assert used <= q.numel() + 12 * 8 * fp8._PACK_NUMBERS + (8 << 20)
