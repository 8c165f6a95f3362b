"""8-bit block-scaled matrices: quantizer, its inverse, products with gradients, and the first half of a gated feed-forward block.

A matrix `[rows, k]` (k a multiple of 16) is a pair of codes `q`, `torch.float8_e4m3fn` `[rows, k]`, and scales `s`, uint8 (exponent
plus 127; 255 is NaN), one for every block of 128:

* `"row"`: 128 columns of a row, in words of four blocks, `[ceil(k/512), rows, 4]` - activations and their gradients where a product sums
  over their columns,
* `"column"`: 128 rows of a column, `[ceil(rows/512), k, 4]` - both operands of a weight's gradient, which sums over the tokens,
* `"square"`: 128 x 128, `[ceil(rows/128), ceil(k/128)]` - weights, which are summed over either way.

A block's scale is the smallest power of two over which its largest magnitude is not above 448, the largest e4m3 number, and not below
2^-127; numbers over the scale are rounded to nearest with ties to even.  A block with an infinity or NaN reads back as NaN.

The gradients are explicit calls, as everything here: none of them takes part in torch's autograd.  The reference has no counterpart.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib
from ._lib import check
from .mx import _expect_output, _expect_sizes, _launched
from .ops import _expect, _on_device, _stream_ptr

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_FP8 = 4
_CODES = torch.float8_e4m3fn
_BLOCKS = {"row": 0, "column": 1, "both": 2, "square": 3}
_ONE_WAY = {b: c for b, c in _BLOCKS.items() if b != "both"}
_ACTIVATIONS = {"silu": 0, "gelu": 1}
_MATMUL, _GATED, _BACKWARD = 0, 1, 2


class _NoFront:
    """Where the native front is missing every call is checked here."""

    @staticmethod
    def _python_way(*args):
        return False

    fp8_quantize = fp8_dequant = fp8_matmul = fp8_matmul_backward = fp8_gated = fp8_gated_backward = _python_way


@functools.lru_cache(maxsize=None)
def _front():
    """The native front (csrc/fast_call.cpp), which checks and launches the common calls, bound to the library."""
    front = _lib.load_fast_call()
    if front is None:
        return _NoFront
    lib = _lib.load()
    front.bind_fp8(*(ctypes.cast(getattr(lib, "tuna_fp8_" + name), ctypes.c_void_p).value for name in
                     ("quantize", "dequant", "matmul", "matmul_backward", "gated", "gated_backward", "workspace_bytes")))
    return front


def _scale_shape(rows: int, k: int, blocks: str):
    if blocks == "square":
        return (-(-rows // 128), -(-k // 128))
    return (-(-k // 512), rows, 4) if blocks == "row" else (-(-rows // 512), k, 4)


def _choice(value, name, choices):
    if value not in choices:
        raise ValueError(f"{name} must be one of {', '.join(map(repr, choices))}, got {value!r}")
    return choices[value]


def _expect_codes(q, s, names, rows, k, blocks, device=None):
    _expect(q, names[0], _CODES, rows * k, device)
    numel = 1
    for d in _scale_shape(rows, k, blocks):
        numel *= d
    _expect(s, names[1], torch.uint8, numel, q.device)


def _expect_16bit(x, name, numel, device=None, dtype=None):
    """The library's type of `x`, checked."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if x.dtype not in (torch.float16, torch.bfloat16) or (dtype is not None and x.dtype != dtype):
        raise TypeError(f"{name} must be {dtype or 'torch.float16 or torch.bfloat16'}, got {x.dtype}")
    _expect(x, name, x.dtype, numel, device)
    return _TYPES[x.dtype]


def _tokens(x, xs, n, k, blocks, device=None):
    """The library's type of the tokens, checked."""
    if xs is not None:
        _expect_codes(x, xs, ("x", "xs"), n, k, blocks, device)
        return _FP8
    return _expect_16bit(x, "x", n * k, device)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _workspace(given, device, call, m, n, k, x_type):
    """The workspace, and its address and size: `given`, or one of this call's own (in stream order, from the pool of the graph that is being
    captured, if one is)."""
    if given is not None:
        _expect(given, "workspace", getattr(given, "dtype", None), given.numel() if isinstance(given, torch.Tensor) else 0, device)
    else:
        need = int(_lib.load().tuna_fp8_workspace_bytes(call, m, n, k, x_type))
        given = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    return given, (0, 0) if given is None else (given.data_ptr(), given.numel() * given.element_size())


def fp8_quantize(x, blocks: str = "row"):
    """`x` (fp16, bf16 or fp32, `[rows, k]`, whose rows may lie apart) -> codes and scales `(q, s)` of that kind of blocks, or, for `"both"`,
    `(q, s, q_column, s_column)` by row and by column in one pass."""
    kind = _choice(blocks, "blocks", _BLOCKS)
    done = _front().fp8_quantize(x, kind)
    if isinstance(done, tuple):
        return done
    _launched(done)
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("x must be a CUDA tensor (there is no CPU path)")
    if x.dtype not in _TYPES:
        raise TypeError(f"x must be torch.float16, torch.bfloat16 or torch.float32, got {x.dtype}")
    if x.dim() != 2 or x.numel() == 0:
        raise ValueError("x must be a [rows, k] tensor with at least one row")
    rows, k = x.shape
    _expect_sizes(rows, k)
    if k % 16:
        raise ValueError(f"k must be a multiple of 16, got {k}")
    stride = k
    if rows == 1:
        if not x.is_contiguous():
            raise ValueError("x must be contiguous")
    elif x.stride(1) != 1 or x.stride(0) < k:
        raise ValueError("the columns of x must be contiguous and its rows must not overlap")
    else:
        stride = x.stride(0)
    out = []
    for b in ("row", "column") if blocks == "both" else (blocks,):
        out += [torch.empty((rows, k), dtype=_CODES, device=x.device), torch.empty(_scale_shape(rows, k, b), dtype=torch.uint8, device=x.device)]
    with _on_device(x.device):
        check(_lib.load().tuna_fp8_quantize(x.data_ptr(), _TYPES[x.dtype], stride, kind, *(t.data_ptr() for t in out), *([0] * (4 - len(out))), rows, k, _stream_ptr(x.device)))
    return tuple(out)


def fp8_dequant(q, s, o, m: int, k: int, blocks: str = "square") -> None:
    """The numbers of codes and scales, rounded once to o's type: o fp16, bf16 or fp32 `[m, k]`."""
    kind = _choice(blocks, "blocks", _ONE_WAY)
    if _launched(_front().fp8_dequant(q, s, o, m, k, kind)):
        return
    _expect_sizes(m, k)
    _expect_codes(q, s, ("q", "s"), m, k, blocks)
    dev = q.device
    _expect_output(o, m * k, dev)
    with _on_device(dev):
        check(_lib.load().tuna_fp8_dequant(q.data_ptr(), s.data_ptr(), kind, o.data_ptr(), _TYPES[o.dtype], m, k, _stream_ptr(dev)))


def fp8_matmul(x, xs, q, s, o, m: int, n: int, k: int, *, workspace=None) -> None:
    """o `[n, m]` (fp16, bf16 or fp32, overwritten) = x `[n, k]` times the transposed matrix of `(q, s)` `[m, k]` (square blocks), fp32 accumulation,
    one rounding; for o in fp32 long sums are made of parts, so that they are as exact as sums in fp32 that round.  x is codes with their scales `xs` (row blocks), or fp16 or bf16 with `xs=None`: the call quantizes it as `fp8_quantize` does.
    m and k multiples of 16.  Enqueued on the current stream of x's device, in whose order it reads and writes; only q and s, up to 64 tokens, count
    as constants and are read while the kernel before still drains, as in `mx_matmul`."""
    if workspace is None and _launched(_front().fp8_matmul(x, xs, q, s, o, m, n, k)):
        return
    _expect_sizes(m, n, k)
    kind = _tokens(x, xs, n, k, "row")
    dev = x.device
    _expect_codes(q, s, ("q", "s"), m, k, "square", dev)
    _expect_output(o, n * m, dev)
    with _on_device(dev):
        _keep, ws = _workspace(workspace, dev, _MATMUL, m, n, k, kind)
        check(_lib.load().tuna_fp8_matmul(x.data_ptr(), kind, _ptr(xs), q.data_ptr(), s.data_ptr(), o.data_ptr(), _TYPES[o.dtype], m, n, k, *ws, _stream_ptr(dev)))


def _expect_gradients(x, xs, q, s, dx, dw, m, n, k, dev):
    """What the gradients that are wanted read and write, checked; the library's type of x."""
    if dx is None and dw is None:
        raise ValueError("dx or dw must be given")
    kind = _FP8
    if dx is not None:
        _expect_codes(q, s, ("q", "s"), m, k, "square", dev)
        _expect_output(dx, n * k, dev)
    if dw is not None:
        kind = _tokens(x, xs, n, k, "column", dev)
        _expect_output(dw, m * k, dev)
    return kind


def _type_of(t) -> int:
    return 0 if t is None else _TYPES[t.dtype]


def fp8_matmul_backward(dy, x, xs, q, s, dx, dw, m: int, n: int, k: int, *, workspace=None) -> None:
    """The gradients of `fp8_matmul` given dy `[n, m]` (fp16 or bf16): dx `[n, k]` = dy times the matrix of `(q, s)`, and dw `[m, k]` = dy
    transposed times x, the gradient of the numbers that the codes stand for.  dx and dw are fp16, bf16 or fp32 and overwritten; None for one that is not
    wanted, and what only it needs may be None then (q and s; x and xs).  dy is quantized by row for dx and by column for dw; x `[n, k]` is
    fp16 or bf16 with `xs=None`, quantized by column, or codes with their scales of column blocks, which a forward pass may have kept
    (`fp8_quantize(x, "both")`).  m and k multiples of 16.  In the order of the current stream."""
    if workspace is None and _launched(_front().fp8_matmul_backward(dy, x, xs, q, s, dx, dw, m, n, k)):
        return
    _expect_sizes(m, n, k)
    dy_type = _expect_16bit(dy, "dy", n * m)
    dev = dy.device
    kind = _expect_gradients(x, xs, q, s, dx, dw, m, n, k, dev)
    with _on_device(dev):
        _keep, ws = _workspace(workspace, dev, _BACKWARD, m, n, k, kind)
        check(_lib.load().tuna_fp8_matmul_backward(dy.data_ptr(), dy_type, _ptr(x), kind, _ptr(xs), _ptr(q), _ptr(s), _ptr(dx), _type_of(dx), _ptr(dw), _type_of(dw), m, n, k,
                                                   *ws, _stream_ptr(dev)))


def fp8_gated(x, xs, q, s, h, f: int, n: int, k: int, activation: str = "silu", *, z=None, workspace=None) -> None:
    """The first half of a gated feed-forward block in one launch: h `[n, f]` (fp16, bf16 or fp32, overwritten) = activation(g) * u, g and u
    `[n, f]` being x `[n, k]` times the transposed first and last f rows of the matrix of `(q, s)` `[2f, k]` (square blocks): gate and up projection,
    one over the other.  x as in `fp8_matmul`, and so are the order of reading and the constants.  activation: `"silu"`, or `"gelu"` in its tanh
    form.  z `[n, 2f]` of h's type (fp16 or bf16) keeps g and u, side by side, for `fp8_gated_backward`; h is made of g and u before they are
    rounded; long sums are made of parts then, and h may be a rounding off from the one without z.  f and k multiples of 16."""
    act = _choice(activation, "activation", _ACTIVATIONS)
    if workspace is None and _launched(_front().fp8_gated(x, xs, q, s, h, f, n, k, act, z)):
        return
    _expect_sizes(2 * f, n, k)
    kind = _tokens(x, xs, n, k, "row")
    dev = x.device
    _expect_codes(q, s, ("q", "s"), 2 * f, k, "square", dev)
    _expect_output(h, n * f, dev)
    if z is not None:
        if h.dtype == torch.float32:
            raise TypeError("with z h must be torch.float16 or torch.bfloat16, got torch.float32")
        _expect_16bit(z, "z", n * 2 * f, dev, h.dtype)
    with _on_device(dev):
        _keep, ws = _workspace(workspace, dev, _GATED, 2 * f, n, k, kind)
        check(_lib.load().tuna_fp8_gated(x.data_ptr(), kind, _ptr(xs), q.data_ptr(), s.data_ptr(), h.data_ptr(), _TYPES[h.dtype], _ptr(z), f, n, k, act, *ws, _stream_ptr(dev)))


def fp8_gated_backward(dh, z, x, xs, q, s, dx, dw, f: int, n: int, k: int, activation: str = "silu", *, workspace=None) -> None:
    """The gradients of `fp8_gated` given dh `[n, f]` and z `[n, 2f]` (fp16 or bf16, one type): those of `fp8_matmul_backward`, dw `[2f, k]`, for
    dy = [dh u activation'(g) | dh activation(g)], which is made and quantized in one pass and never stored in 16 bits: in fp32, as elementary operations
    one after the other give it.  Both gradients are those of z as it was kept, rounded."""
    act = _choice(activation, "activation", _ACTIVATIONS)
    if workspace is None and _launched(_front().fp8_gated_backward(dh, z, x, xs, q, s, dx, dw, f, n, k, act)):
        return
    _expect_sizes(2 * f, n, k)
    kind16 = _expect_16bit(dh, "dh", n * f)
    dev = dh.device
    _expect_16bit(z, "z", n * 2 * f, dev, dh.dtype)
    kind = _expect_gradients(x, xs, q, s, dx, dw, 2 * f, n, k, dev)
    with _on_device(dev):
        _keep, ws = _workspace(workspace, dev, _BACKWARD, 2 * f, n, k, kind)
        check(_lib.load().tuna_fp8_gated_backward(dh.data_ptr(), z.data_ptr(), kind16, _ptr(x), kind, _ptr(xs), _ptr(q), _ptr(s), _ptr(dx), _type_of(dx), _ptr(dw), _type_of(dw),
                                                  f, n, k, act, *ws, _stream_ptr(dev)))


def fp8_pack(codes, scales):
    """A checkpoint's matrix with fp32 scales, codes `torch.float8_e4m3fn` `[rows, k]` and scales fp32 `[ceil(rows/128), ceil(k/128)]` of any value, in
    this package's form: `(q, s)` with square blocks.  Blocks whose scale is a power of two, 2^-127 or above, keep their numbers; the others are quantized
    again, each number off by at most half a step of e4m3 (steps do not go below 2^-136).  A block with an infinity or NaN, or a number above fp32's, is
    NaN.  On any device, a few million numbers at a time."""
    if not isinstance(codes, torch.Tensor) or codes.dtype != _CODES or codes.dim() != 2:
        raise ValueError("codes must be a torch.float8_e4m3fn [rows, k] tensor")
    rows, k = codes.shape
    if not isinstance(scales, torch.Tensor) or scales.dtype != torch.float32 or tuple(scales.shape) != _scale_shape(rows, k, "square"):
        raise ValueError(f"scales must be a torch.float32 {list(_scale_shape(rows, k, 'square'))} tensor")
    q = torch.empty((rows, k), dtype=_CODES, device=codes.device)
    s = torch.empty(_scale_shape(rows, k, "square"), dtype=torch.uint8, device=codes.device)
    blocks = max(1, _PACK_NUMBERS // (128 * max(k, 1)))  # of rows
    for b in range(0, s.shape[0], blocks):
        at = slice(128 * b, 128 * (b + blocks))
        q[at], s[b:b + blocks] = _pack_blocks(codes[at], scales[b:b + blocks])
    return q, s


_PACK_NUMBERS = 1 << 22  # of 64 bits and some of their kind at once: a third of a gigabyte


def _pack_blocks(codes, scales):
    rows, k = codes.shape
    # in 64 bits: the product of a code and a scale is exact, and so is what it becomes over a power of two
    blocks = torch.nn.functional.pad(codes.double(), (0, -k % 128, 0, -rows % 128)).unflatten(0, (-1, 128)).unflatten(2, (-1, 128)) * scales.double()[:, None, :, None]
    largest = blocks.abs().amax((1, 3))
    mantissa, exponent = torch.frexp(largest)
    exponent = torch.where(largest > 0, exponent - 9 + (mantissa > 0.875).int(), -127).clamp(min=-127)  # 0.875 2^9 is 448
    fits = torch.isfinite(largest) & (exponent <= 120)
    exponent = torch.where(fits, exponent, 0)
    y = torch.where(fits[:, None, :, None], blocks, 0.0) * torch.ldexp(torch.ones_like(largest), -exponent)[:, None, :, None]
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y).exponent - 1).clamp(min=-6) - 3)
    q = (torch.round(y / step) * step).flatten(2).flatten(0, 1)[:rows, :k].float().to(_CODES).contiguous()
    return q, torch.where(fits, exponent + 127, 255).to(torch.uint8)
