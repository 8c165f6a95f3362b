"""What is timed of the 8-bit block-scaled operators: the calls that a program built on this package makes, over the range of sizes it makes them at.

A block-scaled matrix `[rows, k]` holds e4m3 codes (`torch.float8_e4m3fn`, row by row) and a power-of-two scale (a byte, exponent
plus 127) for every block of 128: the smallest power of two over which the block's largest magnitude is not above 448, and not below 2^-127.  Blocks are

* "row": 128 columns of a row, bytes in words of four `[ceil(k/512), rows, 4]` - a product's operand whose columns are summed over,
* "column": 128 rows of a column, `[ceil(rows/512), k, 4]` - one whose rows are summed over, as a weight's gradient does with tokens,
* "square": 128 x 128, `[ceil(rows/128), ceil(k/128)]` - weights, which are summed over either way.

A program quantizes weights once.  Serving, a step multiplies activations with them (`fp8_matmul`), and the first half of an MLP is one call:
both projections, the activation and the product (`fp8_gated`).  Training, a step takes the gradients of both as well
(`fp8_matmul_backward`, `fp8_gated_backward`), the weights' being those of the numbers that the codes stand for.

m = output features, f = features of the gated block (its weights are `[2f, k]`, gate first), n = tokens, k = input features.  The sizes are
those of the layers that the repository's tables and benchmark name (hidden 4096 with a 14336-wide MLP, hidden 8192) or generic ones that no
tile size divides.  Weights are normal; activations are normal with a few channels that are twenty times larger, as they are behind a
norm; gradients are small, and some tokens' are all zero, as a padded batch leaves them.
"""

import math
import random

import torch

own = False

MAX_FLOPS = 12 * 14336 * 2048 * 4096       # of the largest listed step
MAX_WEIGHTS = 28672 * 8192                 # of a drawn matrix
MAX_ELEMENTS = 28672 * 4096                # of the largest listed quantization
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4, "fp8": 1 + 1 / 128}
BLOCK = 128


def listed():
    return [
        # the activations of one token on their way into a layer: the smallest call
        {"name": "quantize_1_token", "op": "quantize", "blocks": "row", "n": 1, "k": 4096, "x": "bf16"},
        # a prompt's activations, for the product and for the weight's gradient
        {"name": "quantize_1999_both", "op": "quantize", "blocks": "both", "n": 1999, "k": 14336, "x": "bf16"},
        # a layer's weights after a step of the optimiser, from the copy in 32 bits
        {"name": "quantize_gateup_master", "op": "quantize", "blocks": "square", "n": 28672, "k": 4096, "x": "fp32"},
        # a decode step of one sequence: the smallest layer
        {"name": "decode_1_attn", "op": "matmul", "m": 4096, "n": 1, "k": 4096, "x": "bf16", "o": "bf16"},
        # a decode step of 43 sequences whose activations are codes already, on a layer whose sizes no tile divides
        {"name": "decode_43_ragged", "op": "matmul", "m": 11024, "n": 43, "k": 4112, "x": "fp8", "o": "fp32"},
        # a prompt of a length that no tile divides, hidden size 8192
        {"name": "prefill_777_qkv", "op": "matmul", "m": 10240, "n": 777, "k": 8192, "x": "bf16", "o": "bf16"},
        # gradients of a small layer over a short, odd batch
        {"name": "gradient_301_ragged", "op": "matmul_backward", "m": 1552, "n": 301, "k": 1040, "x": "fp16", "o": "fp16", "dw": "fp32"},
        # gradients of the attention's projections over a 4096-token batch
        {"name": "gradient_4096_qkv", "op": "matmul_backward", "m": 6144, "n": 4096, "k": 4096, "x": "bf16", "o": "bf16", "dw": "bf16"},
        # the first half of an MLP in a decode step of one sequence
        {"name": "gated_1_mlp", "op": "gated", "act": "silu", "f": 14336, "n": 1, "k": 4096, "x": "bf16", "o": "bf16"},
        # the same for a prompt
        {"name": "gated_2000_mlp", "op": "gated", "act": "silu", "f": 14336, "n": 2000, "k": 4096, "x": "bf16", "o": "bf16"},
        # a training step of a small block with the other activation: forward and backward pass
        {"name": "train_333_ragged", "op": "gated_step", "act": "gelu", "f": 1360, "n": 333, "k": 784, "x": "fp16", "o": "fp16", "dw": "fp32"},
        # a training step of a large one: the most work
        {"name": "train_2048_mlp", "op": "gated_step", "act": "silu", "f": 14336, "n": 2048, "k": 4096, "x": "bf16", "o": "bf16", "dw": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _multiple(rng, lo, hi):
    """A multiple of 16; half of the time one of 128, as most layers are."""
    step = 128 if rng.random() < 0.5 else 16
    return max(step, _log_int(rng, lo, hi) // step * step)


def draw(rng):
    """One more case of the ranges above: sizes spread over their logarithm, redrawn until they cost no more than the largest listed ones."""
    while True:
        op = rng.choice(["quantize", "matmul", "matmul", "matmul_backward", "gated", "gated", "gated_step"])
        k = _multiple(rng, 128, 16384)
        case = {"op": op}
        if op == "quantize":
            case.update(blocks=rng.choice(["row", "column", "both", "square"]), n=_log_int(rng, 1, 28672), k=k, x=rng.choice(["fp16", "bf16", "fp32"]))
            if case["n"] * k <= MAX_ELEMENTS:
                return case
            continue
        if op in ("gated", "gated_step"):
            case.update(act=rng.choice(["silu", "gelu"]), f=_multiple(rng, 128, 16384))
        else:
            case["m"] = _multiple(rng, 128, 28672)
        case.update(n=_log_int(rng, 1, 4096), k=k, x=rng.choice(["fp16", "bf16", "fp8"]), o=rng.choice(["fp16", "bf16", "fp32"]))
        if op in ("matmul_backward", "gated_step"):  # of numbers in 16 bits: those are what both passes are given
            case.update(x=rng.choice(["fp16", "bf16"]), dw=rng.choice(["bf16", "fp32"]))
            case["o"] = case["x"]
        if _features(case) * k <= MAX_WEIGHTS and work(case)["flops"] <= MAX_FLOPS:
            return case


def _features(case):
    return 2 * case["f"] if "f" in case else case["m"]


def work(case):
    """Activations, weights, gradients that are given and results once each; two operations per product."""
    n, k, op = case["n"], case["k"], case["op"]
    if op == "quantize":  # read once; codes and scales written and, read back, numbers written, of either way of blocks
        ways = 2 if case["blocks"] == "both" else 1
        return {"bytes": n * k * (BYTES[case["x"]] + ways * (BYTES["fp8"] + BYTES[case["x"]])), "flops": 0}
    rows = _features(case)
    out = case["f"] if "f" in case else rows
    moved = n * k * BYTES[case["x"]] + rows * k
    if op != "matmul_backward":
        moved += n * out * BYTES[case["o"]]
    if op in ("matmul_backward", "gated_step"):
        moved += n * out * BYTES[case["x"]] + n * k * BYTES[case["o"]] + rows * k * BYTES[case["dw"]]
    return {"bytes": moved, "flops": {"matmul": 2, "gated": 2, "matmul_backward": 4, "gated_step": 6}[op] * n * rows * k}


# ---- the format, in 32 bits

def _blocks(x, blocks):
    """`x` [rows, k], padded with zeros, as [blocks of rows, rows, blocks of columns, columns]."""
    r, c = {"row": (1, BLOCK), "column": (BLOCK, 1), "square": (BLOCK, BLOCK)}[blocks]
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % c, 0, -x.shape[0] % r))
    return x.reshape(x.shape[0] // r, r, x.shape[1] // c, c)


def _scale_exponents(x):
    """Of blocks, one scale each: the largest magnitude is m 2^e with m in [1/2, 1), and over 2^(e - 9) it is 512 m."""
    m, e = torch.frexp(x.abs().amax((1, 3), keepdim=True))
    return (e - 9 + (m > 0.875).int()).clamp(min=-127)


def _power_of_two(e, dtype):
    return torch.ldexp(torch.ones_like(e, dtype=dtype), e)


def _round_e4m3(y):
    """To the nearest e4m3 number, ties to the even code: three bits behind the leading one, and steps of 2^-9 below 2^-6."""
    step = _power_of_two((torch.frexp(y).exponent - 1).clamp(min=-6) - 3, y.dtype)
    return torch.round(y / step) * step


def _fake_quantize(x, blocks):
    """The numbers that `x` [rows, k] becomes, in 32 bits."""
    b = _blocks(x.float(), blocks)
    scale = _power_of_two(_scale_exponents(b), torch.float32)
    y = _round_e4m3(b / scale) * scale
    return y.reshape(y.shape[0] * y.shape[1], -1)[:x.shape[0], :x.shape[1]]


def _pack(x, blocks):
    """Codes and scales of `x` [rows, k] in the package's layout; row or square blocks."""
    b = _blocks(x.float(), blocks)
    e = _scale_exponents(b)
    y = _round_e4m3(b / _power_of_two(e, torch.float32))
    q = y.reshape(y.shape[0] * y.shape[1], -1)[:x.shape[0], :x.shape[1]].contiguous().to(torch.float8_e4m3fn)
    s = (e + 127).to(torch.uint8).reshape(e.shape[0], e.shape[2])
    if blocks == "row":
        s = torch.nn.functional.pad(s, (0, -s.shape[1] % 4)).unflatten(1, (-1, 4)).transpose(0, 1).contiguous()
    return q, s


def _numbers(q, s, blocks, dtype):
    """The numbers of codes and scales; row or square blocks."""
    if blocks == "row":
        s = s.transpose(0, 1).flatten(1).repeat_interleave(BLOCK, 1)
    else:
        s = s.repeat_interleave(BLOCK, 0).repeat_interleave(BLOCK, 1)
    return q.to(dtype) * _power_of_two(s[:q.shape[0], :q.shape[1]].int() - 127, dtype)


def _gate(g, act):
    """What the activation multiplies its argument with, and the derivative of the product of both."""
    if act == "silu":
        p, dp = g, torch.ones_like(g)
    else:  # gelu in its tanh form: (1 + tanh(y)) / 2 is the logistic function of 2 y
        c = 2 * math.sqrt(2 / math.pi)
        p, dp = c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g ** 2)
    s = 1 / (1 + torch.exp(-p))
    return s, s + g * s * (1 - s) * dp


# ---- what a program has in hand

def _activations(gen, n, k):
    x = torch.randn((n, k), generator=gen, device="cuda")
    heavy = torch.randint(0, k, (max(1, k // 500),), generator=gen, device="cuda")
    x[:, heavy] *= 20
    return x


def _gradient(gen, n, m):
    dy = torch.randn((n, m), generator=gen, device="cuda").mul_(n ** -0.5)
    dy[n - n // 10:] = 0  # what pads the batch
    return dy


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, k, op = case["n"], case["k"], case["op"]
    x_type = TYPES.get(case["x"])
    state = {"case": case}
    if op == "quantize":
        x = torch.randn((n, k), generator=gen, device="cuda").mul_(k ** -0.5) if case["blocks"] == "square" else _activations(gen, n, k)
        state["x"] = x.to(x_type)
        state["o"] = [torch.empty((n, k), device="cuda", dtype=x_type) for _ in range(2 if case["blocks"] == "both" else 1)]
        return state
    rows = _features(case)
    out = case["f"] if "f" in case else rows
    state["q"], state["s"] = _pack(torch.randn((rows, k), generator=gen, device="cuda").mul_(k ** -0.5), "square")
    x = _activations(gen, n, k)
    state["x"], state["xs"] = _pack(x, "row") if x_type is None else (x.to(x_type), None)
    if op != "matmul_backward":
        state["o"] = torch.zeros((n, out), device="cuda", dtype=TYPES[case["o"]])
    if op in ("matmul_backward", "gated_step"):
        state["dy"] = _gradient(gen, n, out).to(x_type)
        state["dx"] = torch.zeros((n, k), device="cuda", dtype=TYPES[case["o"]])
        state["dw"] = torch.zeros((rows, k), device="cuda", dtype=TYPES[case["dw"]])
    if op == "gated_step":
        state["z"] = torch.zeros((n, rows), device="cuda", dtype=x_type)  # the projections, kept for the backward pass
    return state


# ---- one pass

def run(state):
    case = state["case"]
    op, n, k = case["op"], case["n"], case["k"]
    if own:
        return _run_own(state, case, op, n, k)
    x = state["x"]
    if op == "quantize":
        ways = ["row", "column"] if case["blocks"] == "both" else [case["blocks"]]
        return [_fake_quantize(x, b).to(x.dtype) for b in ways]
    w = _numbers(state["q"], state["s"], "square", torch.float32)
    if op != "matmul_backward":
        y = (_fake_quantize(x, "row") if state["xs"] is None else _numbers(x, state["xs"], "row", torch.float32)) @ w.transpose(0, 1)
        if op == "matmul":
            return y.to(TYPES[case["o"]])
        g, u = y.split(case["f"], 1)
        h = (g * _gate(g, case["act"])[0] * u).to(TYPES[case["o"]])
        if op == "gated":
            return h
        # the backward pass has the projections as they were kept
        g, u = y.to(x.dtype).float().split(case["f"], 1)
        sigma, derivative = _gate(g, case["act"])
        dh = state["dy"].float()
        dy = torch.cat((dh * u * derivative, dh * g * sigma), 1)
    else:
        dy = state["dy"]
    dx = _fake_quantize(dy, "row") @ w
    dw = _fake_quantize(dy, "column").transpose(0, 1) @ _fake_quantize(x, "column")
    dx, dw = dx.to(TYPES[case["o"]]), dw.to(TYPES[case["dw"]])
    return [dx, dw] if op == "matmul_backward" else [h, dx, dw]


def _run_own(state, case, op, n, k):
    import tuna_b200

    x = state["x"]
    if op == "quantize":
        blocks, o = case["blocks"], state["o"]
        codes = tuna_b200.fp8_quantize(x, blocks)
        if blocks == "both":
            tuna_b200.fp8_dequant(codes[0], codes[1], o[0], n, k, "row")
            tuna_b200.fp8_dequant(codes[2], codes[3], o[1], n, k, "column")
        else:
            tuna_b200.fp8_dequant(*codes, o[0], n, k, blocks)
        return o
    q, s, xs = state["q"], state["s"], state["xs"]
    if op == "matmul":
        tuna_b200.fp8_matmul(x, xs, q, s, state["o"], case["m"], n, k)
        return state["o"]
    if op == "gated":
        tuna_b200.fp8_gated(x, xs, q, s, state["o"], case["f"], n, k, case["act"])
        return state["o"]
    if op == "matmul_backward":
        tuna_b200.fp8_matmul_backward(state["dy"], x, None, q, s, state["dx"], state["dw"], case["m"], n, k)
        return [state["dx"], state["dw"]]
    tuna_b200.fp8_gated(x, xs, q, s, state["o"], case["f"], n, k, case["act"], z=state["z"])
    tuna_b200.fp8_gated_backward(state["dy"], state["z"], x, None, q, s, state["dx"], state["dw"], case["f"], n, k, case["act"])
    return [state["o"], state["dx"], state["dw"]]


# ---- the definition in 64 bits

def _exact_numbers(x, blocks):
    """Block by block: the scale from the bits of the largest magnitude, numbers between neighbours of e4m3 by their distance."""
    v = x.double()
    r, c = {"row": (1, BLOCK), "column": (BLOCK, 1), "square": (BLOCK, BLOCK)}[blocks]
    largest = torch.nn.functional.max_pool2d(torch.nn.functional.pad(v.abs(), (0, -v.shape[1] % c, 0, -v.shape[0] % r))[None], (r, c))[0]
    bits = largest.view(torch.int64)
    exponent = (bits >> 52) - 1023 - 8 + ((bits & ((1 << 52) - 1)) > (3 << 50)).long()  # 1.75 2^8 is 448
    scale = ((exponent.clamp(min=-127) + 1023) << 52).view(torch.float64)
    scale = scale.repeat_interleave(r, 0).repeat_interleave(c, 1)[:v.shape[0], :v.shape[1]]
    y = v.abs() / scale
    step = ((((y.view(torch.int64) >> 52) - 1023).clamp(min=-6) - 3 + 1023) << 52).view(torch.float64)
    below = torch.floor(y / step)
    rest = y / step - below
    up = (rest > 0.5) | ((rest == 0.5) & (below.long() % 2 == 1))
    return torch.sign(v) * (below + up) * step * scale


def _exact_decoded(q, s, blocks):
    """A matrix's numbers from the bits of its codes (sign, four of exponent, three of mantissa) and scales."""
    c = q.view(torch.uint8).long()
    exponent, mantissa = (c >> 3) & 15, (c & 7).double()
    v = torch.where(exponent > 0, (1 + mantissa / 8) * torch.exp2((exponent - 7).double()), mantissa * 2.0 ** -9)
    v = torch.where(c >= 128, -v, v)
    row = torch.arange(q.shape[0], device=q.device)[:, None]
    col = torch.arange(q.shape[1], device=q.device)[None]
    byte = s[col // 512, row, col // BLOCK % 4] if blocks == "row" else s[row // BLOCK, col // BLOCK]
    return v * ((byte.long() - 127 + 1023) << 52).view(torch.float64)


def _exact_activation(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    t = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * g * g)


def exact(case, seed):
    state = prepare(case, seed)
    op, x = case["op"], state["x"]
    if op == "quantize":
        return [_exact_numbers(x, b) for b in (["row", "column"] if case["blocks"] == "both" else [case["blocks"]])]
    w = _exact_decoded(state["q"], state["s"], "square")
    if op != "matmul_backward":
        y = torch.einsum("nk,mk->nm", _exact_numbers(x, "row") if state["xs"] is None else _exact_decoded(x, state["xs"], "row"), w)
        if op == "matmul":
            return y
        f = case["f"]
        h = _exact_activation(y[:, :f], case["act"])[0] * y[:, f:]
        if op == "gated":
            return h
        z = y.to(x.dtype).double()
        value, derivative = _exact_activation(z[:, :f], case["act"])
        dh = state["dy"].double()
        dy = torch.cat((dh * z[:, f:] * derivative, dh * value), 1)
    else:
        dy = state["dy"]
    dx = torch.einsum("nm,mk->nk", _exact_numbers(dy, "row"), w)
    dw = torch.einsum("nm,nk->mk", _exact_numbers(dy, "column"), _exact_numbers(x, "column"))
    return [dx, dw] if op == "matmul_backward" else [h, dx, dw]
