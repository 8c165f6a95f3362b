"""8-bit block-scaled operators, what needs no GPU: the oracle against the format's definition, scales, packing, and refusals."""

import ctypes
import re
from pathlib import Path

import numpy as np
import pytest
import torch

import tuna_b200
from oracle import fp8_oracle as fo
from tuna_b200 import fp8


def test_oracle_magnitudes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double().numpy()
    mine = fo.decode(codes.numpy()[None], np.array([[127, 127]], dtype=np.uint8), "row")[0]
    assert np.array_equal(mine, want, equal_nan=True)


def test_oracle_rounds_to_nearest_with_ties_to_even():
    grid = fo.MAGNITUDES
    middle = (grid[1:] + grid[:-1]) / 2
    for v, lower in ((middle, np.arange(126)), (np.nextafter(middle, 0), None), (np.nextafter(middle, 1e9), None)):
        want = lower + lower % 2 if lower is not None else np.arange(126) + (v > middle)
        assert np.array_equal(fo.encode(v), want) and np.array_equal(fo.encode(-v), want | 128)
    assert fo.encode(np.array([448.0, 464.0, 1e30])).tolist() == [126] * 3


def test_oracle_scales():
    x = np.zeros((1, 128 * 9))
    for b, v in enumerate([448.0, np.nextafter(448.0, 1e9), 1.0, 1.75, np.nextafter(1.75, 2), 2.0 ** -140, 0.0, np.inf, np.nan]):
        x[0, 128 * b + 5] = v
    _, s = fo.quantize(x, "row")
    assert s[0].tolist() == [127, 128, 119, 119, 120, 0, 0, 255, 255]


def test_layout_of_scale_words():
    s = np.arange(1, 16, dtype=np.uint8).reshape(3, 5)  # three rows of five blocks
    w = fo.pack(s, "row")
    assert w.shape == (2, 3, 4) and w[0, 1].tolist() == [6, 7, 8, 9] and w[1, 2].tolist() == [15, 0, 0, 0]
    w = fo.pack(s.T.copy(), "column")  # five blocks of rows, three columns
    assert w.shape == (2, 3, 4) and w[0, 1].tolist() == [6, 7, 8, 9] and w[1, 2].tolist() == [15, 0, 0, 0]
    for blocks, shape in (("row", (2, 300, 4)), ("column", (1, 528, 4)), ("square", (3, 5))):
        assert fp8._scale_shape(300, 528, blocks) == shape


@pytest.mark.parametrize("rows,k", [(1, 16), (128, 128), (200, 272), (300, 144)])
def test_pack_keeps_numbers_where_scales_are_powers_of_two(rows, k):
    rng = np.random.default_rng(rows)
    codes = rng.integers(0, 127, (rows, k), dtype=np.uint8) | (rng.integers(0, 2, (rows, k), dtype=np.uint8) << 7)
    e = rng.integers(-30, 30, (-(-rows // 128), -(-k // 128)))
    q, s = tuna_b200.fp8_pack(torch.from_numpy(codes).view(torch.float8_e4m3fn), torch.from_numpy(np.ldexp(1.0, e).astype(np.float32)))
    want = fo.decode(codes, (e + 127).astype(np.uint8), "square")
    assert np.array_equal(fo.decode(q.view(torch.uint8).numpy(), s.numpy(), "square"), want)
    # any other scale: what the quantizer makes of the numbers
    f = (np.ldexp(1.0, e) * rng.uniform(1, 2, e.shape)).astype(np.float32)
    q, s = tuna_b200.fp8_pack(torch.from_numpy(codes).view(torch.float8_e4m3fn), torch.from_numpy(f))
    v = fo.decode(codes, np.full(e.shape, 127, dtype=np.uint8), "square") * fo.spread(f.astype(np.float64), "square", rows, k)
    assert np.array_equal(fo.decode(q.view(torch.uint8).numpy(), s.numpy(), "square"), fo.numbers(v, "square"))


def test_pack_of_what_is_no_number():
    codes = torch.zeros(1, 384, dtype=torch.uint8)
    codes[0, 3] = 0x7f
    codes[0, 130] = 56  # 1.0
    q, s = tuna_b200.fp8_pack(codes.view(torch.float8_e4m3fn), torch.tensor([[1.0, float("inf"), 1.0]]))
    assert s.tolist() == [[255, 255, 0]] and not q.view(torch.uint8).any()


def test_pack_refuses():
    q = torch.zeros(4, 16, dtype=torch.float8_e4m3fn)
    for args in ((q.view(torch.uint8), torch.ones(1, 1)), (q, torch.ones(1, 2)), (q, torch.ones(1, 1).double()), (q[None], torch.ones(1, 1))):
        with pytest.raises(ValueError):
            tuna_b200.fp8_pack(*args)


def _calls():
    """Every entry point with tensors of the right types and sizes, on the CPU."""
    q = torch.zeros(32, 16, dtype=torch.float8_e4m3fn)
    s = torch.zeros(1, 1, dtype=torch.uint8)
    x, y, h = (torch.zeros(2, c, dtype=torch.bfloat16) for c in (16, 32, 16))
    return {
        "quantize": lambda **kw: tuna_b200.fp8_quantize(kw.get("x", x), kw.get("blocks", "row")),
        "dequant": lambda **kw: tuna_b200.fp8_dequant(q, s, torch.zeros(32, 16), kw.get("m", 32), kw.get("k", 16), kw.get("blocks", "square")),
        "matmul": lambda **kw: tuna_b200.fp8_matmul(kw.get("x", x), None, q, s, y, kw.get("m", 32), kw.get("n", 2), kw.get("k", 16)),
        "backward": lambda **kw: tuna_b200.fp8_matmul_backward(y, kw.get("x", x), None, q, s, kw.get("dx", x), kw.get("dw", torch.zeros(32, 16)), kw.get("m", 32), kw.get("n", 2), kw.get("k", 16)),
        "gated": lambda **kw: tuna_b200.fp8_gated(kw.get("x", x), None, q, s, h, kw.get("m", 16), kw.get("n", 2), kw.get("k", 16), kw.get("act", "silu")),
        "gated_backward": lambda **kw: tuna_b200.fp8_gated_backward(h, y, kw.get("x", x), None, q, s, kw.get("dx", x), kw.get("dw", torch.zeros(32, 16)), kw.get("m", 16), kw.get("n", 2),
                                                                    kw.get("k", 16), kw.get("act", "silu")),
    }


@pytest.mark.parametrize("name", list(_calls()))
def test_tensors_off_the_gpu_are_refused(name):
    with pytest.raises(ValueError, match="CUDA"):
        _calls()[name]()


@pytest.mark.parametrize("name", ["dequant", "matmul", "backward", "gated", "gated_backward"])
def test_sizes_of_more_than_32_bits_are_refused(name):
    for size in ("m", "k") if name == "dequant" else ("m", "n", "k"):
        with pytest.raises(ValueError, match="2147483647"):
            _calls()[name](**{size: 2 ** 32 + 16})


def test_unknown_names_are_refused():
    for name, kw in (("quantize", {"blocks": "tile"}), ("dequant", {"blocks": "both"}), ("gated", {"act": "relu"}), ("gated_backward", {"act": None})):
        with pytest.raises(ValueError, match="must be one of"):
            _calls()[name](**kw)


def test_argument_validation_needs_no_gpu(tuna_lib):
    buf = ctypes.create_string_buffer(4096 + 64)
    base = (ctypes.addressof(buf) + 63) & ~63
    p, odd, odder = (ctypes.c_void_p(base + i) for i in (0, 8, 2))
    big = 1 << 40

    def qz(x=p, x_type=0, stride=32, blocks=0, q=p, s=p, q2=None, s2=None, rows=2, k=32):
        return tuna_lib.tuna_fp8_quantize(x, x_type, stride, blocks, q, s, q2, s2, rows, k, None)

    assert qz(x=None) == -1 and qz(q=None) == -1 and qz(s=None) == -1 and qz(blocks=2) == -1 and qz(blocks=2, q2=p) == -1
    assert qz(rows=0) == -2 and qz(k=24) == -2 and qz(k=0) == -2 and qz(stride=16) == -2 and qz(rows=-1) == -2
    assert qz(x_type=3) == -5 and qz(x_type=4) == -5 and qz(blocks=4) == -5 and qz(blocks=-1) == -5
    assert qz(x=odd) == -3 and qz(q=odd) == -3 and qz(stride=36) == -3 and qz(s=odder) == -3 and qz(blocks=2, q2=odd, s2=p) == -3
    assert qz(k=8388624, stride=8388624) == -9 and qz(rows=(1 << 31) - 1) == -9

    def dq(q=p, s=p, blocks=3, o=p, o_type=0, rows=2, k=32):
        return tuna_lib.tuna_fp8_dequant(q, s, blocks, o, o_type, rows, k, None)

    assert dq(q=None) == -1 and dq(s=None) == -1 and dq(o=None) == -1 and dq(k=24) == -2 and dq(rows=0) == -2
    assert dq(blocks=2) == -5 and dq(blocks=4) == -5 and dq(o_type=4) == -5 and dq(q=odd) == -3 and dq(o=odd) == -3
    assert dq(k=8388624) == -9 and dq(rows=(1 << 31) - 1) == -9

    def mm(x=p, x_type=4, xs=p, q=p, s=p, o=p, o_type=0, m=64, n=1, k=64, ws=p, ws_bytes=big):
        return tuna_lib.tuna_fp8_matmul(x, x_type, xs, q, s, o, o_type, m, n, k, ws, ws_bytes, None)

    def gt(x=p, x_type=4, xs=p, q=p, s=p, o=p, o_type=0, z=p, m=64, n=1, k=64, act=0, ws=p, ws_bytes=big):
        return tuna_lib.tuna_fp8_gated(x, x_type, xs, q, s, o, o_type, z, m, n, k, act, ws, ws_bytes, None)

    for call in (mm, gt):
        assert call(x=None) == -1 and call(xs=None) == -1 and call(q=None) == -1 and call(s=None) == -1 and call(o=None) == -1
        assert call(m=56) == -2 and call(n=0) == -2 and call(k=56) == -2 and call(k=0) == -2 and call(m=-16) == -2
        assert call(x_type=2) == -5 and call(x_type=3) == -5 and call(o_type=4) == -5
        assert call(x=odd) == -3 and call(xs=odder) == -3 and call(q=odd) == -3 and call(o=odd) == -3 and call(ws=odd) == -3
        assert call(x_type=0, n=33, ws=None) == -4 and call(x_type=0, n=33, ws_bytes=33 * 64) == -4
        assert call(m=8388624) == -9 and call(k=8388624) == -9 and call(n=(1 << 31) - 1) == -9
    assert gt(act=2) == -5 and gt(o_type=2) == -5 and gt(z=odd) == -3  # z has 16 bits

    def bw(dy=p, dy_type=0, x=p, x_type=1, xs=None, q=p, s=p, dx=p, dx_type=0, dw=p, dw_type=2, m=64, n=3, k=64, ws=p, ws_bytes=big):
        return tuna_lib.tuna_fp8_matmul_backward(dy, dy_type, x, x_type, xs, q, s, dx, dx_type, dw, dw_type, m, n, k, ws, ws_bytes, None)

    def gb(dy=p, dy_type=0, z=p, x=p, x_type=1, xs=None, q=p, s=p, dx=p, dx_type=0, dw=p, dw_type=2, m=64, n=3, k=64, act=0, ws=p, ws_bytes=big):
        return tuna_lib.tuna_fp8_gated_backward(dy, z, dy_type, x, x_type, xs, q, s, dx, dx_type, dw, dw_type, m, n, k, act, ws, ws_bytes, None)

    for call in (bw, gb):
        assert call(dy=None) == -1 and call(dx=None, dw=None) == -1 and call(q=None) == -1 and call(s=None) == -1 and call(x=None) == -1 and call(x_type=4) == -1
        assert call(m=56) == -2 and call(n=0) == -2 and call(k=56) == -2
        assert call(dy_type=2) == -5 and call(dy_type=4) == -5 and call(dx_type=4) == -5 and call(dw_type=3) == -5 and call(x_type=2) == -5
        assert call(dy=odd) == -3 and call(dx=odd) == -3 and call(dw=odd) == -3 and call(x=odd) == -3 and call(q=odd) == -3 and call(ws=odd) == -3 and call(x_type=4, xs=odder) == -3
        assert call(ws=None) == -4 and call(ws_bytes=3 * 64) == -4
        assert call(m=8388624) == -9 and call(n=(1 << 31) - 1) == -9
    assert gb(z=None) == -1 and gb(z=odd) == -3 and gb(act=2) == -5


def test_workspace_sizes(tuna_lib):
    ws = tuna_lib.tuna_fp8_workspace_bytes
    assert ws(0, 64, 33, 64, 4) == 0 and ws(1, 64, 33, 64, 4) == 0
    assert ws(0, 64, 33, 64, 0) >= 33 * (64 + 4) and ws(1, 64, 33, 64, 1) >= 33 * (64 + 4)
    assert ws(0, 4096, 1, 4096, 0) == 0  # a token that the product quantizes itself
    # dy by row and by column, x by column unless it is codes
    assert ws(2, 64, 700, 128, 0) >= 700 * (64 + 4) + 700 * 64 + 2 * 4 * 64 + 700 * 128 + 2 * 4 * 128
    assert ws(2, 64, 700, 128, 0) > ws(2, 64, 700, 128, 4) >= 700 * (64 + 4) + 700 * 64 + 2 * 4 * 64
    for bad in ((0, 56, 1, 64, 0), (0, 64, 0, 64, 0), (0, 64, 1, 8, 0), (3, 64, 1, 64, 0), (-1, 64, 1, 64, 0), (0, 64, 1, 8388624, 0)):
        assert ws(*bad) == 0


def test_numbers_match_the_header():
    header = (Path(__file__).resolve().parents[1] / "include" / "tuna_b200.h").read_text()
    values = {n: int(v) for n, v in re.findall(r"(TUNA_[A-Z0-9_]+) = (\d)", header)}
    assert {values["TUNA_FP8_" + n.upper()] for n in fp8._BLOCKS} == set(fp8._BLOCKS.values()) and values["TUNA_FP8_SQUARE"] == fp8._BLOCKS["square"]
    assert values["TUNA_FP8"] == fp8._FP8 and (values["TUNA_SILU"], values["TUNA_GELU"]) == (fp8._ACTIVATIONS["silu"], fp8._ACTIVATIONS["gelu"])
    assert [values["TUNA_FP8_" + n] for n in ("MATMUL", "GATED", "BACKWARD")] == [fp8._MATMUL, fp8._GATED, fp8._BACKWARD]
    assert fp8._TYPES == {torch.float16: values["TUNA_FP16"], torch.bfloat16: values["TUNA_BF16"], torch.float32: values["TUNA_FP32"]}


def test_what_other_kernels_write_is_not_loaded_through_the_read_only_path():
    """These kernels start before the ones that write their inputs have ended."""
    for path in (Path(fp8.__file__).parent / "csrc").glob("fp8_*"):
        source = re.sub(r"//[^\n]*", "", path.read_text())
        assert ".nc" not in source and "__ldg(" not in source and "__restrict__" not in source, path.name


@pytest.mark.parametrize("kind", ["silu", "gelu"])
def test_oracle_activation_against_differences(kind):
    g = np.linspace(-8, 8, 161)
    value, slope = fo.activation(g, kind)
    h = 1e-5
    assert np.allclose((fo.activation(g + h, kind)[0] - fo.activation(g - h, kind)[0]) / (2 * h), slope, atol=1e-9)
    t = torch.from_numpy(g)
    want = torch.nn.functional.silu(t) if kind == "silu" else torch.nn.functional.gelu(t, approximate="tanh")
    assert np.allclose(value, want.numpy(), atol=1e-15)
