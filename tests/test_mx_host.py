"""Microscaled 4-bit operators, what needs no GPU: the oracle against the format's table, the layout, and refusals."""

import ctypes

import numpy as np
import pytest
import torch

import tuna_b200
from oracle import mx_oracle as mxo
from tuna_b200 import mx


def test_oracle_magnitudes_and_ties():
    assert mxo.MAGNITUDES.tolist() == [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    ties = {0.25: 0, 0.75: 2, 1.25: 2, 1.75: 4, 2.5: 4, 3.5: 6, 5.0: 6}  # to the even code
    for v, code in ties.items():
        assert mxo.encode(np.array([v]))[0] == code
        assert mxo.encode(np.array([-v]))[0] == code | 8
        assert mxo.encode(np.array([np.nextafter(v, 10)]))[0] == (code if code % 2 == 0 and mxo.MAGNITUDES[code] > v else code + 1)
    assert mxo.encode(np.array([6.0, 7.9, 1e9])).tolist() == [7, 7, 7]


def test_oracle_scales():
    x = np.zeros((1, 32 * 6))
    for b, v in enumerate([1.0, 7.999, 2.0 ** -130, 0.0, np.inf, np.nan]):
        x[0, 32 * b] = v
    _, s = mxo.quantize(x)
    assert s[0].tolist() == [125, 127, 0, 0, 255, 255]


@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (8, 256), (5, 288), (2, 4128)])
def test_pack_puts_codes_and_scales_where_the_layout_says(rows, k):
    rng = np.random.default_rng(k)
    codes = rng.integers(0, 16, (rows, k), dtype=np.uint8)
    scales = rng.integers(0, 256, (rows, k // 32), dtype=np.uint8)
    q, s = mxo.pack(codes, scales)
    back = mxo.unpack(q, s, k)
    assert np.array_equal(back[0], codes) and np.array_equal(back[1], scales)
    q2, s2 = tuna_b200.mx_pack(torch.from_numpy(codes[:, 0::2] | codes[:, 1::2] << 4), torch.from_numpy(scales))
    assert np.array_equal(q2.numpy(), q) and np.array_equal(s2.numpy(), s)
    q3, s3 = tuna_b200.mx_pack(torch.from_numpy(np.stack([codes[:, 0::2] | codes[:, 1::2] << 4] * 2)), torch.from_numpy(np.stack([scales] * 2)))
    assert q3.shape == (2, *q.shape) and np.array_equal(q3[1].numpy(), q) and np.array_equal(s3[1].numpy(), s)


def test_pack_refuses():
    u8 = dict(dtype=torch.uint8)
    with pytest.raises(ValueError):
        tuna_b200.mx_pack(torch.zeros(4, 16), torch.zeros(4, 1, **u8))
    with pytest.raises(ValueError):
        tuna_b200.mx_pack(torch.zeros(4, 16, **u8), torch.zeros(4, 2, **u8))
    with pytest.raises(ValueError):
        tuna_b200.mx_pack(torch.zeros(4, 16, **u8), torch.zeros(5, 1, **u8))


def test_tensors_off_the_gpu_are_refused():
    u8 = dict(dtype=torch.uint8)
    q, s = torch.zeros(1, 8, 128, **u8), torch.zeros(2, 8, 4, **u8)
    o = torch.zeros(1, 8)
    for call in (lambda: tuna_b200.mx_quantize(torch.zeros(8, 256)), lambda: tuna_b200.mx_dequant(q, s, torch.zeros(8, 256), 8, 256),
                 lambda: tuna_b200.mx_matmul(torch.zeros(1, 256).half(), None, q, s, o, 8, 1, 256),
                 lambda: tuna_b200.mx_matmul_grouped(torch.zeros(1, 256).half(), None, q[None], s[None], torch.zeros(2, dtype=torch.int32), o, 8, 1, 256)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        tuna_b200.mx_matmul(torch.zeros(1, 256), None, q, s, o, 8, 1, 256)


def test_sizes_of_more_than_32_bits_are_refused():
    t, big = torch.zeros(1, dtype=torch.uint8), 2 ** 32
    for call in (lambda: tuna_b200.mx_matmul(t, t, t, t, t, 8, 1, big + 32), lambda: tuna_b200.mx_matmul(t, t, t, t, t, big + 8, 1, 32),
                 lambda: tuna_b200.mx_matmul(t, t, t, t, t, 8, big + 1, 32), lambda: tuna_b200.mx_dequant(t, t, t, 1, big + 32),
                 lambda: tuna_b200.mx_matmul_grouped(t, t, t, t, t, t, 8, big, 32)):
        with pytest.raises(ValueError, match="2147483647"):
            call()


def test_argument_validation_needs_no_gpu(tuna_lib):
    buf = ctypes.create_string_buffer(4096 + 64)
    base = (ctypes.addressof(buf) + 63) & ~63
    p, odd = ctypes.c_void_p(base), ctypes.c_void_p(base + 4)
    qz = tuna_lib.tuna_mx_quantize
    assert qz(None, 0, 32, p, p, 1, 32, 1, None) == -1
    assert qz(p, 0, 32, p, None, 1, 32, 1, None) == -1
    assert qz(p, 0, 32, p, p, 0, 32, 1, None) == -2
    assert qz(p, 0, 48, p, p, 1, 48, 1, None) == -2          # k % 32
    assert qz(p, 0, 32, p, p, 1, 32, 0, None) == -2          # no matrix
    assert qz(p, 0, 31, p, p, 2, 32, 1, None) == -2          # rows overlap
    assert qz(p, 3, 32, p, p, 1, 32, 1, None) == -5          # codes are not numbers
    assert qz(p, 0, 36, p, p, 2, 32, 1, None) == -3          # rows not 16-byte aligned
    assert qz(odd, 0, 32, p, p, 1, 32, 1, None) == -3
    assert qz(p, 0, 1 << 30, p, p, 1 << 30, 1 << 30, 1, None) == -9
    dq = tuna_lib.tuna_mx_dequant
    assert dq(p, None, p, 0, 1, 32, 1, None) == -1
    assert dq(p, p, p, 0, 1, 16, 1, None) == -2
    assert dq(p, p, p, 7, 1, 32, 1, None) == -5
    assert dq(p, p, odd, 0, 1, 32, 1, None) == -3
    big = 1 << 40

    def mm(x=p, x_type=3, xs=p, q=p, s=p, o=p, o_type=0, m=64, n=1, k=64, ws=p, ws_bytes=big):
        return tuna_lib.tuna_mx_matmul(x, x_type, xs, q, s, o, o_type, m, n, k, ws, ws_bytes, None)

    assert mm(x=None) == -1 and mm(xs=None) == -1 and mm(q=None) == -1 and mm(s=None) == -1 and mm(o=None) == -1
    assert mm(m=60) == -2 and mm(n=0) == -2 and mm(k=48) == -2 and mm(k=0) == -2 and mm(m=-8) == -2
    assert mm(x_type=2) == -5 and mm(x_type=4) == -5 and mm(o_type=3) == -5
    assert mm(x=odd) == -3 and mm(xs=ctypes.c_void_p(base + 2)) == -3 and mm(q=odd) == -3 and mm(s=odd) == -3 and mm(o=odd) == -3 and mm(ws=odd) == -3
    # tokens in 16 bits that a launch of their own quantizes: room for their codes and scales
    need = tuna_lib.tuna_mx_workspace_bytes(64, 33, 64, 0, 0)
    assert need >= 33 * (128 + 4) and tuna_lib.tuna_mx_workspace_bytes(64, 33, 64, 0, 3) == 0
    assert mm(x_type=0, n=33, ws=None) == -4 and mm(x_type=0, n=33, ws_bytes=need - 1) == -4

    # nothing is launched - not the tokens' quantizer either - for what the product refuses
    assert mm(x_type=0, m=8, n=(1 << 31) - 1, k=1024, ws_bytes=1 << 60) in (-7, -9)

    # sizes that rounded up to a whole tile would no longer have 32 bits, more columns than a grid has chunks for
    long = (1 << 31) - 32
    for type_ in (0, 3):
        assert mm(x_type=type_, m=8, n=(1 << 31) - 1, k=32, ws_bytes=1 << 60) == -9 and mm(x_type=type_, m=long, k=32) == -9
        for k in (67107840 + 32, long):
            assert mm(x_type=type_, m=8, k=k, ws_bytes=1 << 60) == -9
    assert qz(p, 0, 32, p, p, (1 << 31) - 1, 32, 1, None) == -9 and dq(p, p, p, 0, (1 << 31) - 1, 32, 1, None) == -9
    for k in (67107840 + 32, long):
        assert qz(p, 0, k, p, p, 1, k, 1, None) == -9 and dq(p, p, p, 0, 1, k, 1, None) == -9
        assert tuna_lib.tuna_mx_workspace_bytes(8, 1, k, 0, 0) == 0

    def grouped(offsets=p, experts=2, n=4, x_type=3, ws_bytes=big):
        return tuna_lib.tuna_mx_matmul_grouped(p, x_type, p, p, p, offsets, p, 0, 64, n, 64, experts, p, ws_bytes, None)

    assert grouped(offsets=None) == -1
    assert grouped(experts=0) == -2
    assert grouped(experts=1025) == -9
    assert grouped(offsets=ctypes.c_void_p(base + 2)) == -3
    assert grouped(x_type=1, ws_bytes=0) == -4
    assert grouped(n=0) == 0 and grouped(n=-1) == -2
    assert tuna_lib.tuna_mx_workspace_bytes(60, 33, 64, 0, 0) == 0
    assert tuna_lib.tuna_mx_workspace_bytes(64, 1, 64, 1025, 0) == 0


def test_types_match_the_header():
    import re
    from pathlib import Path

    header = (Path(__file__).resolve().parents[1] / "include" / "tuna_b200.h").read_text()
    values = {n: int(v) for n, v in re.findall(r"(TUNA_(?:FP16|BF16|FP32|MXFP4)) = (\d)", header)}
    assert values == {"TUNA_FP16": mx._TYPES[torch.float16], "TUNA_BF16": mx._TYPES[torch.bfloat16], "TUNA_FP32": mx._TYPES[torch.float32], "TUNA_MXFP4": mx._MXFP4}


def test_tokens_are_not_loaded_through_the_read_only_path():
    """Kernels that quantize a product's tokens start before the kernel that writes these has ended, and PTX allows ld.global.nc (and
    __ldg) only for what nobody writes while the kernel lives."""
    import re
    from pathlib import Path

    source = re.sub(r"//[^\n]*", "", (Path(mx.__file__).parent / "csrc" / "mx_format.cuh").read_text())
    loads = re.findall(r"void load\(const \w+ \*p\) \{([^}]*)\}", source)
    assert len(loads) == 3
    for load in loads:
        assert set(re.findall(r"(\w+)\(p", load)) == {"mx_load_u4"}
    assert ".nc" not in source and "ldg" not in source


def test_as_many_output_features_as_are_accepted(tuna_lib):
    """A plan that rounds m up to whole tiles on every SM must not pass 32 bits for any m that is not refused: the tokens of a call this small are
    quantized by the product itself, whatever m is."""
    most = (1 << 31) - 1024
    for m in (8 * 1000, 1 << 30, most - 128 * 148, most - 18936, most - 8, most):
        for n in (1, 2, 16):
            assert tuna_lib.tuna_mx_workspace_bytes(m, n, 32, 0, 0) == 0, (m, n)
    assert tuna_lib.tuna_mx_workspace_bytes(most, 17, 32, 0, 0) == 17 * (128 + 4)
    assert tuna_lib.tuna_mx_workspace_bytes(most + 8, 1, 32, 0, 0) == 0
    buf = ctypes.create_string_buffer(4096 + 64)
    p = ctypes.c_void_p((ctypes.addressof(buf) + 63) & ~63)
    assert tuna_lib.tuna_mx_matmul(p, 3, p, p, p, p, 0, most + 8, 1, 32, p, 1 << 40, None) == -9


def test_row_scales_are_not_loaded_through_the_read_only_path():
    """The codebook kernels start early as well, and absmax follows ordinary stream order."""
    import re
    from pathlib import Path

    for path in (Path(mx.__file__).parent / "csrc").glob("gemm_*.cu"):
        source = re.sub(r"//[^\n]*", "", path.read_text())
        assert "absmax" in source and "__ldg(" not in source, path.name
