"""Microscaled quantizer and its inverse on the GPU, bit for bit against the oracle in 64 bits."""

import numpy as np
import pytest
import torch

import tuna_b200
from tests.gpu_util import Guarded
from oracle import mx_oracle as mxo
from tuna_b200 import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def neighbour(v, step):
    """The next number of positive `v`'s type, up or down."""
    ints = torch.int32 if v.dtype == torch.float32 else torch.int16
    return (v.view(ints) + step).view(v.dtype)


def check(x):
    """Codes and scales of x, and what they read back as, in every type."""
    q, s = tuna_b200.mx_quantize(x)
    codes, scales = mxo.quantize(x.double().cpu().numpy())
    qr, sr = mxo.pack(codes, scales)
    assert np.array_equal(s.cpu().numpy(), sr)
    live = np.repeat(scales != 255, 32, axis=-1)  # a NaN block's codes do not matter
    got = mxo.unpack(q.cpu().numpy(), s.cpu().numpy(), x.shape[1])[0]
    assert np.array_equal(got[live], codes[live])
    pad = q.cpu().numpy().reshape(q.shape[0], q.shape[1], -1).transpose(1, 0, 2).reshape(q.shape[1], -1)[:, x.shape[1] // 2:]
    assert not pad.any(), "codes behind the last column are zero"
    numbers = torch.from_numpy(mxo.decode(codes, scales))
    for t in TYPES:
        hold = Guarded(x.numel() * t.itemsize, t, x.shape)
        tuna_b200.mx_dequant(q, s, hold.view, *x.shape)
        torch.cuda.synchronize()
        assert hold.guards_intact()
        want = numbers.to(t)  # 64 bits -> t: one rounding, as from fp32, which holds the numbers exactly
        assert torch.equal(torch.nan_to_num(hold.view.cpu().float(), nan=12345.0), torch.nan_to_num(want.float(), nan=12345.0))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 4096), (2, 64), (7, 96), (8, 256), (9, 288), (17, 4128), (64, 1024), (129, 2080), (300, 32)])
def test_rows_and_widths(rows, k, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows * 1000 + k)
    x = torch.randn((rows, k), generator=gen, device="cuda") * torch.exp2(torch.randint(-6, 7, (rows, 1), generator=gen, device="cuda").float())
    check(x.to(dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_border_between_codes(dtype):
    """Every midpoint of two magnitudes and its neighbours in the type, both signs, under scales from small to large."""
    rows = []
    for e in (-20, -14, -3, 0, 5, 12) if dtype == torch.float16 else (-130, -127, -126, -100, 0, 60, 124):
        borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=torch.float64) * 2.0 ** e
        b = borders.to(dtype)
        row = torch.zeros(64, dtype=dtype)
        row[0], row[32] = 4 * 2.0 ** e, -7.5 * 2.0 ** e if e < 13 or dtype != torch.float16 else -6 * 2.0 ** e
        row[1:9], row[9:17], row[17:25] = b, neighbour(b, -1), -b
        row[33:41], row[41:49], row[49:57] = b, neighbour(b, 1), -neighbour(b, -1)
        rows.append(row)
    check(torch.stack(rows).cuda())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_extremes(dtype):
    info = torch.finfo(dtype)
    x = torch.zeros(6, 256, dtype=dtype)
    x[0, :32] = info.max
    x[0, 32] = -info.max
    x[1, 5], x[1, 70] = info.tiny, info.smallest_normal * 0.75   # subnormals
    x[2, 3], x[2, 40], x[2, 100], x[2, 101] = float("inf"), float("-inf"), float("nan"), 1.0
    x[3] = -0.0
    x[4, 200:] = torch.linspace(-1, 1, 56).to(dtype)
    x[5] = info.max / 2
    check(x.cuda())


def test_rows_that_lie_apart_and_views():
    base = torch.randn(40, 3 * 512, device="cuda", dtype=torch.bfloat16)
    for view in (base[:, 512:1024], base[3:21, 512:800], base[::2, :512], base[5:6, :512]):
        if view.shape[0] == 1:
            view = view.contiguous()
        q, s = tuna_b200.mx_quantize(view)
        q2, s2 = tuna_b200.mx_quantize(view.contiguous())
        assert torch.equal(q, q2) and torch.equal(s, s2)


def test_sets_of_matrices():
    x = torch.randn(3, 13, 416, device="cuda", dtype=torch.float16)
    q, s = tuna_b200.mx_quantize(x)
    o = torch.empty(3, 13, 416, device="cuda", dtype=torch.float32)
    tuna_b200.mx_dequant(q, s, o, 13, 416)
    for i in range(3):
        qi, si = tuna_b200.mx_quantize(x[i])
        assert torch.equal(q[i], qi) and torch.equal(s[i], si)
        one = torch.empty(13, 416, device="cuda")
        tuna_b200.mx_dequant(qi, si, one, 13, 416)
        assert torch.equal(o[i], one)


def test_every_scale_byte_reads_back():
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    q, s = (torch.from_numpy(a).cuda() for a in mxo.pack(codes, scales))
    numbers = torch.from_numpy(mxo.decode(codes, scales))
    for t in TYPES:
        o = torch.empty(256, 32, device="cuda", dtype=t)
        tuna_b200.mx_dequant(q, s, o, 256, 32)
        assert torch.equal(torch.nan_to_num(o.cpu().float(), nan=12345.0), torch.nan_to_num(numbers.to(t).float(), nan=12345.0))


def test_more_than_2_31_elements():
    rows, k = 68000, 32768
    x = torch.zeros(rows, k, device="cuda", dtype=torch.bfloat16)
    at = torch.tensor([0, 33333, 65535, 65536, 67997, 67998, 67999], device="cuda")
    x[at] = torch.randn(len(at), k, device="cuda", dtype=torch.bfloat16)
    q, s = tuna_b200.mx_quantize(x)
    small = tuna_b200.mx_quantize(x[at])
    assert torch.equal(q[:, at], small[0]) and torch.equal(s[:, at], small[1])
    o = torch.full((rows, k), 7.0, device="cuda", dtype=torch.bfloat16)
    tuna_b200.mx_dequant(q, s, o, rows, k)
    want = torch.empty(len(at), k, device="cuda", dtype=torch.bfloat16)
    tuna_b200.mx_dequant(*small, want, len(at), k)
    assert torch.equal(o[at], want)
    o[at] = 0
    assert not o.any()


def test_nothing_is_written_behind_the_last_row():
    lib = _lib.load()
    x = torch.randn(5, 160, device="cuda", dtype=torch.float16)
    q, s = Guarded(5 * 128, torch.uint8, (1, 5, 128)), Guarded(2 * 5 * 4, torch.uint8, (2, 5, 4))
    assert lib.tuna_mx_quantize(x.data_ptr(), 0, 160, q.view.data_ptr(), s.view.data_ptr(), 5, 160, 1, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert q.guards_intact() and s.guards_intact()
    q2, s2 = tuna_b200.mx_quantize(x)
    assert torch.equal(q.view, q2) and torch.equal(s.view, s2)


@pytest.mark.parametrize("rows", [1, 3])
def test_as_many_columns_as_there_may_be(rows):
    k = 67107840
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device="cuda", dtype=torch.float16)
    x = levels[torch.randint(0, 16, (rows, k), device="cuda", dtype=torch.uint8).int()]
    x[:, ::32] = 6  # every block's scale is 1: nothing is rounded
    q, s = tuna_b200.mx_quantize(x)
    back = torch.empty_like(x)
    tuna_b200.mx_dequant(q, s, back, rows, k)
    assert torch.equal(back, x) and (s == 127).all()


def test_refusals():
    x = torch.randn(8, 256, device="cuda")
    for bad in (x[:, :40], x.t(), x[:, ::2], x[None].expand(2, 8, 256), x.view(-1), x[:0]):
        with pytest.raises(ValueError):
            tuna_b200.mx_quantize(bad)
    with pytest.raises(TypeError):
        tuna_b200.mx_quantize(x.to(torch.int32))
    with pytest.raises(tuna_b200.TunaError):  # rows not on 16 bytes
        tuna_b200.mx_quantize(torch.randn(8, 130, device="cuda")[:, :128])
    with pytest.raises(ValueError, match="2147483647"):  # ctypes would make 32 of it
        tuna_b200.mx_quantize(torch.empty(1, 2 ** 32 + 32, dtype=torch.float16, device="cuda"))
    q, s = tuna_b200.mx_quantize(x)
    with pytest.raises(TypeError):
        tuna_b200.mx_dequant(q, s, torch.empty(8, 256, device="cuda", dtype=torch.float64), 8, 256)
    with pytest.raises(ValueError):
        tuna_b200.mx_dequant(q, s, torch.empty(8, 255, device="cuda"), 8, 256)
    with pytest.raises(ValueError):
        tuna_b200.mx_dequant(q, s[:1], torch.empty(8, 256, device="cuda"), 8, 256)
