"""The quantizer of 8-bit block-scaled matrices and its inverse on the GPU: codes, scales and numbers bit for bit as the oracle's."""

import numpy as np
import pytest
import torch

import tuna_b200
from oracle import fp8_oracle as fo
from tests.fp8_util import codes_tensor, numpy64, random_matrix
from tests.gpu_util import Guarded

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
WAYS = ["row", "column", "both", "square"]


def check_codes(x, blocks, x64=None):
    """What `fp8_quantize` gives for x, against the oracle."""
    out = tuna_b200.fp8_quantize(x, blocks)
    x64 = numpy64(x) if x64 is None else x64
    for i, way in enumerate(("row", "column") if blocks == "both" else (blocks,)):
        codes, scales = fo.quantize(x64, way)
        q, s = out[2 * i], out[2 * i + 1]
        assert q.dtype == torch.float8_e4m3fn and tuple(q.shape) == x64.shape
        assert np.array_equal(s.cpu().numpy(), fo.pack(scales, way)), way
        assert np.array_equal(q.view(torch.uint8).cpu().numpy(), codes), way
    return out


@pytest.mark.parametrize("blocks", WAYS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,k", [(1, 16), (1, 4096), (3, 144), (16, 512), (127, 128), (128, 256), (129, 1040), (513, 272), (1100, 640), (5, 14336)])
def test_quantize(rows, k, dtype, blocks):
    gen = torch.Generator(device="cuda").manual_seed(rows * k)
    x = torch.randn(rows, k, generator=gen, device="cuda") * torch.exp(4 * torch.randn(rows, 1, generator=gen, device="cuda"))
    x[:, k // 2] *= 50
    check_codes(x.to(dtype), blocks)


@pytest.mark.parametrize("blocks", WAYS)
def test_every_number_of_16_bits(blocks):
    """All fp16 numbers but infinities and NaN, which lie in an order that puts large and small ones in one block."""
    bits = np.random.default_rng(1).permutation(65536).astype(np.uint16)
    x = bits.view(np.float16).reshape(256, 256)
    x = np.where(np.isfinite(x), x, np.float16(0))
    check_codes(torch.from_numpy(x).cuda(), blocks)


@pytest.mark.parametrize("blocks", WAYS)
def test_scales_at_their_borders(blocks):
    """Largest magnitudes at and around 448 times a power of two, the smallest scale, subnormal numbers, zeros and the largest numbers of fp32."""
    x = np.zeros((256, 256), dtype=np.float32)
    for i in range(128):
        x[i, 3 * (i % 40)] = np.float32(448.0) * np.float32(2.0) ** (i - 64)
        x[128 + i, 5] = np.nextafter(np.float32(448.0) * np.float32(2.0) ** (i - 64), np.float32(np.inf))
    x[:64, 200] = np.float32(2.0) ** -149 * np.arange(1, 65)
    x[64:128, 130] = np.finfo(np.float32).max
    x[128:, 128:] = np.float32(2.0) ** -125
    check_codes(torch.from_numpy(x).cuda(), blocks)


@pytest.mark.parametrize("blocks", WAYS)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_blocks_with_infinities_and_nan(dtype, bad, blocks):
    x = torch.randn(300, 400, device="cuda").to(dtype)
    x[7, 3] = x[299, 399] = x[130, 200] = bad
    out = check_codes(x, blocks)
    way = "row" if blocks == "both" else blocks
    o = torch.empty(300, 400, device="cuda")
    tuna_b200.fp8_dequant(out[0], out[1], o, 300, 400, way)
    r, c = fo.SHAPES[way]
    spoilt = fo.spread(fo.largest((~torch.isfinite(x)).double().cpu().numpy(), way), way, 300, 400) > 0
    assert np.array_equal(torch.isnan(o).cpu().numpy(), spoilt)


@pytest.mark.parametrize("blocks", WAYS)
def test_rows_that_lie_apart(blocks):
    wide = torch.randn(200, 400, device="cuda", dtype=torch.bfloat16)
    x = wide[:, 16:16 + 272]
    out = tuna_b200.fp8_quantize(x, blocks)
    for a, b in zip(out, tuna_b200.fp8_quantize(x.contiguous(), blocks)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("blocks", ["row", "column", "square"])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,k", [(1, 16), (5, 1040), (130, 272), (513, 144), (1030, 512)])
def test_dequant(rows, k, dtype, blocks):
    (q, s), x = random_matrix(rows, k, blocks, rows + k)
    hold = Guarded(rows * k * dtype.itemsize, dtype, (rows, k))
    tuna_b200.fp8_dequant(q, s, hold.view, rows, k, blocks)
    torch.cuda.synchronize()
    assert hold.guards_intact()
    assert torch.equal(hold.view.cpu(), torch.from_numpy(x).to(dtype))


def test_dequant_of_every_code_and_scale():
    codes = np.tile(np.arange(256, dtype=np.uint8), (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 2, 1)
    o = torch.empty(256, 256, device="cuda")
    tuna_b200.fp8_dequant(codes_tensor(codes), torch.from_numpy(fo.pack(scales, "row")).cuda(), o, 256, 256, "row")
    with np.errstate(over="ignore"):
        want = fo.decode(codes, scales, "row").astype(np.float32)
    assert np.array_equal(o.cpu().numpy(), want, equal_nan=True)


def test_nothing_outside_the_results_is_written():
    rows, k = 150, 208
    from tuna_b200 import _lib

    x = torch.randn(rows, k, device="cuda", dtype=torch.float16)
    lib, stream = _lib.load(), torch.cuda.current_stream().cuda_stream
    for blocks, code in (("row", 0), ("column", 1), ("square", 3)):
        from tuna_b200 import fp8

        shape = fp8._scale_shape(rows, k, blocks)
        q, s = Guarded(rows * k, torch.uint8, (rows, k)), Guarded(int(np.prod(shape)), torch.uint8, shape)
        assert lib.tuna_fp8_quantize(x.data_ptr(), 0, k, code, q.view.data_ptr(), s.view.data_ptr(), 0, 0, rows, k, stream) == 0
        torch.cuda.synchronize()
        assert q.guards_intact() and s.guards_intact()


def test_more_elements_than_2_31():
    rows, k = 140000, 16384
    x = torch.zeros(rows, k, device="cuda", dtype=torch.bfloat16)
    x[rows - 3:] = torch.randn(3, k, device="cuda").bfloat16()
    x[rows - 3:, 100] = 300.0
    for blocks in ("row", "column", "square"):
        q, s = tuna_b200.fp8_quantize(x, blocks)
        o = torch.empty(rows, k, device="cuda", dtype=torch.bfloat16)
        tuna_b200.fp8_dequant(q, s, o, rows, k, blocks)
        first = (rows - 3) // 128 * 128
        tail = numpy64(x[first:])
        assert np.array_equal(numpy64(o[first:]), numpy64(torch.from_numpy(fo.numbers(tail, blocks)).bfloat16()))
        assert not o[:first].any()
        del q, s, o


def test_refusals():
    x = torch.zeros(4, 32, device="cuda", dtype=torch.bfloat16)
    for bad in (x[:, :24], x.t(), x[0], x[:0], x.view(torch.int16), x.expand(4, 32)[:, ::2]):
        with pytest.raises((ValueError, TypeError)):
            tuna_b200.fp8_quantize(bad)
    with pytest.raises(tuna_b200.TunaError):
        tuna_b200.fp8_quantize(torch.zeros(4, 40, device="cuda", dtype=torch.bfloat16)[:, 4:36])  # rows not on 16 bytes
    q, s = tuna_b200.fp8_quantize(x)
    o = torch.empty(4, 32, device="cuda")
    tuna_b200.fp8_dequant(q, s, o, 4, 32, "row")
    for args in ((q, s, o, 4, 16, "row"), (q, s, o, 4, 32, "square"), (q.view(torch.uint8), s, o, 4, 32, "row"), (q, s, o.double(), 4, 32, "row"), (q, s, o[:3], 4, 32, "row")):
        with pytest.raises((ValueError, TypeError)):
            tuna_b200.fp8_dequant(*args)


@pytest.mark.parametrize("blocks", WAYS)
def test_captured_and_replayed(blocks):
    x = torch.randn(300, 528, device="cuda", dtype=torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tuna_b200.fp8_quantize(x, blocks)
    for _ in range(2):
        x.copy_(torch.randn(300, 528, device="cuda") * 7)
        graph.replay()
        for a, b in zip(out, tuna_b200.fp8_quantize(x, blocks)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
