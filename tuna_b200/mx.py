"""Microscaled 4-bit (OCP MXFP4) matrices: quantizer, its inverse, and products in which both operands have 4 bits.

A matrix `[rows, k]` (k a multiple of 32) is a pair of uint8 tensors: codes `q` `[ceil(k/256), rows, 128]`, column 2j of a
256-column chunk in the low nibble of byte j and 2j+1 in the high one, and scales `s` `[ceil(k/128), rows, 4]`, a byte
(exponent plus 127; 255 is NaN) for every 32 columns.  What lies behind column k in the last chunk is zero.  A set of
experts' matrices has a leading dimension.  Column ranges are views of the leading dimension of chunks and words where they start at a
multiple of 256 and end at one, or at the matrix's end.  A range that ends inside a chunk has the columns behind it there instead of
zeros, and has to be copied and cleared: products take them in, as many as the number of tokens makes them.

The reference has no counterpart: its one 4-bit format is the codebook of `matmul`.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._lib import check
from .ops import _expect, _on_device, _stream_ptr

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_MXFP4 = 3


class _NoFront:
    """Where the native front is missing every call is checked here."""

    @staticmethod
    def _python_way(*args):
        return False

    mx_quantize = mx_dequant = mx_matmul = mx_matmul_grouped = _python_way


@functools.lru_cache(maxsize=None)
def _front():
    """The native front (csrc/fast_call.cpp), which checks and launches the common calls, bound to the library."""
    front = _lib.load_fast_call()
    if front is None:
        return _NoFront
    lib = _lib.load()
    front.bind_mx(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in
                    ("tuna_mx_quantize", "tuna_mx_dequant", "tuna_mx_matmul", "tuna_mx_matmul_grouped", "tuna_mx_workspace_bytes")))
    return front


def _launched(done) -> bool:
    """Whether the front has made the call; an error of the launch itself is raised."""
    if done is not False and done is not True:
        check(done)
    return done is True


def _code_shape(rows: int, k: int):
    return (-(-k // 256), rows, 128)


def _scale_shape(rows: int, k: int):
    return (-(-k // 128), rows, 4)


def _expect_sizes(*sizes):
    """The library's sizes have 32 bits, and ctypes would cut longer ones down to them."""
    if max(sizes) > 0x7fffffff:
        raise ValueError(f"sizes must not be above 2147483647, got {max(sizes)}")


def _numel(shape) -> int:
    return shape[0] * shape[1] * shape[2]


def _expect_codes(q, s, names, rows, k, device=None, matrices=1):
    _expect(q, names[0], torch.uint8, matrices * _numel(_code_shape(rows, k)), device)
    _expect(s, names[1], torch.uint8, matrices * _numel(_scale_shape(rows, k)), q.device)


def _expect_output(o, numel, device):
    if not isinstance(o, torch.Tensor):
        raise TypeError("o must be a torch.Tensor")
    if o.dtype not in _TYPES:
        raise TypeError(f"o must be torch.float16, torch.bfloat16 or torch.float32, got {o.dtype}")
    _expect(o, "o", o.dtype, numel, device)


def _workspace(given, device, *shape_and_type):
    """Address and size of the workspace: `given`, or one of this call's own (in stream order, from the pool of the graph that is being captured,
    if one is)."""
    if given is not None:
        _expect(given, "workspace", getattr(given, "dtype", None), given.numel() if isinstance(given, torch.Tensor) else 0, device)
    else:
        need = int(_lib.load().tuna_mx_workspace_bytes(*shape_and_type))
        given = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    return given, (0, 0) if given is None else (given.data_ptr(), given.numel() * given.element_size())


def mx_quantize(x):
    """`x` (fp16, bf16 or fp32; `[rows, k]`, whose rows may lie apart, or contiguous `[matrices, rows, k]`) -> codes and scales
    `(q, s)`.  A block's scale is 2^(floor(log2(largest magnitude)) - 2), not below 2^-127; numbers over the scale are
    rounded to nearest with ties to even and saturate at 6.  A block with an infinity or NaN reads back as NaN."""
    done = _front().mx_quantize(x)
    if isinstance(done, tuple):
        return done
    _launched(done)
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (there is no CPU path)")
    if x.dtype not in _TYPES:
        raise TypeError(f"x must be torch.float16, torch.bfloat16 or torch.float32, got {x.dtype}")
    if x.dim() not in (2, 3) or x.numel() == 0:
        raise ValueError("x must be a [rows, k] or [matrices, rows, k] tensor with at least one row")
    rows, k = x.shape[-2:]
    _expect_sizes(rows, k)
    if k % 32:
        raise ValueError(f"k must be a multiple of 32, got {k}")
    stride = k
    if x.dim() == 3 or rows == 1:
        if not x.is_contiguous():
            raise ValueError("x must be contiguous")
    elif x.stride(1) != 1 or x.stride(0) < k:
        raise ValueError("the columns of x must be contiguous and its rows must not overlap")
    else:
        stride = x.stride(0)
    lead = tuple(x.shape[:-2])
    q = torch.empty(lead + _code_shape(rows, k), dtype=torch.uint8, device=x.device)
    s = torch.empty(lead + _scale_shape(rows, k), dtype=torch.uint8, device=x.device)
    with _on_device(x.device):
        check(_lib.load().tuna_mx_quantize(x.data_ptr(), _TYPES[x.dtype], stride, q.data_ptr(), s.data_ptr(), rows, k, lead[0] if lead else 1, _stream_ptr(x.device)))
    return q, s


def mx_dequant(q, s, o, m: int, k: int) -> None:
    """The numbers of codes and scales, rounded once to o's type: o fp16, bf16 or fp32 `[m, k]`.  With a leading dimension of q, s
    and o, all its matrices."""
    if _launched(_front().mx_dequant(q, s, o, m, k)):
        return
    _expect_sizes(m, k)
    dev = q.device if isinstance(q, torch.Tensor) else None
    matrices = q.shape[0] if isinstance(q, torch.Tensor) and q.dim() == 4 else 1
    _expect_codes(q, s, ("q", "s"), m, k, dev, matrices)
    _expect_output(o, matrices * m * k, dev)
    with _on_device(dev):
        check(_lib.load().tuna_mx_dequant(q.data_ptr(), s.data_ptr(), o.data_ptr(), _TYPES[o.dtype], m, k, matrices, _stream_ptr(dev)))


def _tokens(x, xs, n, k):
    """The library's type of the tokens, checked."""
    if xs is not None:
        _expect_codes(x, xs, ("x", "xs"), n, k)
        return _MXFP4
    if not isinstance(x, torch.Tensor):
        raise TypeError("x must be a torch.Tensor")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"x must be torch.float16 or torch.bfloat16, or codes with their scales xs, got {x.dtype}")
    _expect(x, "x", x.dtype, n * k)
    return _TYPES[x.dtype]


def mx_matmul(x, xs, q, s, o, m: int, n: int, k: int, *, workspace=None) -> None:
    """o `[n, m]` (fp16, bf16 or fp32, overwritten) = x `[n, k]` times the transposed matrix of `(q, s)` `[m, k]`, fp32 accumulation,
    one rounding.  x is codes with their scales `xs`, or fp16 or bf16 with `xs=None`: the call quantizes it as
    `mx_quantize` does.  m a multiple of 8, k of 32.  Enqueued on the current stream of x's device, in whose order it reads and writes; only
    q and s, up to 64 tokens, count as constants and are read while the kernel before still drains.  A kernel that writes them right
    before such a call must not let its dependents start early (`mx_quantize` does not); behind one that does, put a copy that is not a
    kernel in between, or synchronise."""
    if workspace is None and _launched(_front().mx_matmul(x, xs, q, s, o, m, n, k)):
        return
    _expect_sizes(m, n, k)
    kind = _tokens(x, xs, n, k)
    dev = x.device
    _expect_codes(q, s, ("q", "s"), m, k, dev)
    _expect_output(o, n * m, dev)
    lib = _lib.load()
    with _on_device(dev):
        _keep, ws = _workspace(workspace, dev, m, n, k, 0, kind)
        check(lib.tuna_mx_matmul(x.data_ptr(), kind, 0 if xs is None else xs.data_ptr(), q.data_ptr(), s.data_ptr(), o.data_ptr(), _TYPES[o.dtype], m, n, k,
                                 *ws, _stream_ptr(dev)))


def mx_matmul_grouped(x, xs, q, s, offsets, o, m: int, n: int, k: int, *, workspace=None) -> None:
    """`mx_matmul` for the experts of a mixture, whose tokens lie expert by expert: rows offsets[e] up to offsets[e + 1] of x are
    multiplied with matrix e of `q` `[experts, ceil(k/256), m, 128]` and `s`.  `offsets` int32 `[experts + 1]`, not decreasing (one that is less
    than one before it counts as that one), stays on
    the device (a router's cumulative counts): nothing waits for it on the host.  x and o have n rows, which may be more than
    offsets[experts]: rows of o that no expert has are left as they were.  n = 0 is nothing to do.  All that it reads, q and s too, follows the
    order of the stream."""
    if workspace is None and _launched(_front().mx_matmul_grouped(x, xs, q, s, offsets, o, m, n, k)):
        return
    _expect_sizes(m, n, k)
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise ValueError("q must be a [experts, ceil(k/256), m, 128] tensor")
    experts = q.shape[0]
    kind = _tokens(x, xs, n, k)
    dev = x.device
    _expect_codes(q, s, ("q", "s"), m, k, dev, experts)
    _expect(offsets, "offsets", torch.int32, experts + 1, dev)
    _expect_output(o, n * m, dev)
    if n == 0:
        return
    lib = _lib.load()
    with _on_device(dev):
        _keep, ws = _workspace(workspace, dev, m, n, k, experts, kind)
        check(lib.tuna_mx_matmul_grouped(x.data_ptr(), kind, 0 if xs is None else xs.data_ptr(), q.data_ptr(), s.data_ptr(), offsets.data_ptr(), o.data_ptr(),
                                         _TYPES[o.dtype], m, n, k, experts, *ws, _stream_ptr(dev)))


def mx_pack(codes, scales):
    """Row-major codes uint8 `[.., rows, k/2]` (column 2j in the low nibble of byte j) and scale bytes uint8 `[.., rows, k/32]`, as
    checkpoints have them, in this package's layout: `(q, s)`.  On any device."""
    for t, name in ((codes, "codes"), (scales, "scales")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.dim() not in (2, 3):
            raise ValueError(f"{name} must be a uint8 [rows, ..] or [matrices, rows, ..] tensor")
    if codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != 16 * scales.shape[-1]:
        raise ValueError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} are not of one matrix: 16 bytes of codes go with a byte of scales")
    q = torch.nn.functional.pad(codes, (0, -codes.shape[-1] % 128)).unflatten(-1, (-1, 128)).transpose(-3, -2).contiguous()
    s = torch.nn.functional.pad(scales, (0, -scales.shape[-1] % 4)).unflatten(-1, (-1, 4)).transpose(-3, -2).contiguous()
    return q, s
