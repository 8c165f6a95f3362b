"""What is timed of the microscaled 4-bit operators: the calls that a program built on this package makes, over the range of sizes it makes them at.

A microscaled (MXFP4) matrix holds 4-bit floating-point codes (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and one
power-of-two scale (e8m0) for every 32 columns of a row.  A serving program quantizes its weights once, and in every step

* quantizes activations and, where another kernel wants numbers, reads codes back (`mx_quantize`, `mx_dequant`),
* multiplies them with a layer's weights (`mx_matmul`), codes of both or activations that the call quantizes itself,
* multiplies tokens that lie expert by expert with each expert's weights (`mx_matmul_grouped`).

m = output features, n = tokens, k = reduction length.  Codes are kept in chunks of 256 columns, `q` uint8
`[ceil(k/256), rows, 128]` with column 2j of a chunk in the low nibble of byte j and 2j+1 in the high one, scales in words
of four, `s` uint8 `[ceil(k/128), rows, 4]` (exponent plus 127); what lies behind column k is zero.  Experts' weights have
a leading dimension.

The sizes are those of the layers that the repository's tables and benchmark name (hidden 4096 with a 14336-wide MLP, hidden
8192, eight experts) or generic ones that no tile size divides.  Weights are normal; activations are normal with a few channels
that are twenty times larger, as they are behind a norm.
"""

import random

import torch

own = False

MAX_FLOPS = 2 * 57344 * 4096 * 8192        # of the largest listed product
MAX_WEIGHTS = 8 * 28672 * 4096             # of the largest listed set of experts
MAX_ELEMENTS = 57344 * 8192                # of the largest listed quantization
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4, "mx": 17 / 32}


def listed():
    return [
        # the activations of one token on their way into a layer: the smallest call
        {"name": "quantize_1_token", "op": "quantize", "n": 1, "k": 4096, "x": "bf16", "o": "bf16"},
        # a prompt's activations in front of a down projection
        {"name": "quantize_1999_prompt", "op": "quantize", "n": 1999, "k": 14336, "x": "bf16", "o": "bf16"},
        # a layer's weights when a model is loaded, and back for a kernel that wants numbers
        {"name": "quantize_gateup", "op": "quantize", "n": 57344, "k": 8192, "x": "fp16", "o": "fp16"},
        # a master copy in 32 bits, of a width that ends inside a chunk
        {"name": "quantize_master", "op": "quantize", "n": 5000, "k": 8224, "x": "fp32", "o": "fp32"},
        # a decode step of one sequence: the smallest layer, from activations in 16 bits
        {"name": "decode_1_attn", "op": "matmul", "m": 4096, "n": 1, "k": 4096, "x": "bf16", "o": "bf16"},
        # a decode step of 16 sequences: gate+up projection
        {"name": "decode_16_gateup", "op": "matmul", "m": 28672, "n": 16, "k": 4096, "x": "fp16", "o": "fp16"},
        # a step of 43 sequences whose activations are codes already, on a layer whose sizes no tile divides
        {"name": "decode_43_ragged", "op": "matmul", "m": 11000, "n": 43, "k": 4128, "x": "mx", "o": "fp32"},
        # a prompt of a length that no tile divides, hidden size 8192
        {"name": "prefill_777_qkv", "op": "matmul", "m": 10240, "n": 777, "k": 8192, "x": "bf16", "o": "bf16"},
        # the largest product: gate+up of hidden size 8192 over a 4096-token prompt chunk
        {"name": "prefill_4096_gateup", "op": "matmul", "m": 57344, "n": 4096, "k": 8192, "x": "mx", "o": "bf16"},
        # gate+up of eight experts in a decode step of 16 sequences with two experts each
        {"name": "experts_32_gateup", "op": "grouped", "experts": 8, "m": 28672, "n": 32, "k": 4096, "routing": 3, "behind": 0, "x": "bf16", "o": "bf16"},
        # down projections of eight experts for a prompt, in a buffer with room behind the last token
        {"name": "experts_1500_down", "op": "grouped", "experts": 8, "m": 4096, "n": 1500, "k": 14336, "routing": 5, "behind": 51, "x": "mx", "o": "bf16"},
        # many small experts, some of them without a token
        {"name": "experts_64_small", "op": "grouped", "experts": 64, "m": 2048, "n": 150, "k": 1024, "routing": 8, "behind": 0, "x": "fp16", "o": "fp16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _multiple(rng, lo, hi, unit):
    """A multiple of `unit`; half of the time one of 256, as most layers are."""
    step = 256 if rng.random() < 0.5 else unit
    return max(step, _log_int(rng, lo, hi) // step * step)


def draw(rng):
    """One more case of the ranges above: sizes spread over their logarithm, redrawn until they cost no more than the largest listed ones."""
    while True:
        op = rng.choice(["quantize", "matmul", "matmul", "grouped"])
        k = _multiple(rng, 256, 28672, 32)
        if op == "quantize":
            t = rng.choice(["fp16", "bf16", "fp32"])
            case = {"op": op, "n": _log_int(rng, 1, 57344), "k": k, "x": t, "o": t}
            if case["n"] * k <= MAX_ELEMENTS:
                return case
            continue
        m = _multiple(rng, 256, 57344, 8)
        case = {"op": op, "m": m, "n": _log_int(rng, 1, 4096), "k": k, "x": rng.choice(["fp16", "bf16", "mx"]), "o": rng.choice(["fp16", "bf16", "fp32"])}
        if op == "grouped":
            case.update(experts=_log_int(rng, 2, 64), routing=rng.randint(0, 1 << 20), behind=rng.choice([0, rng.randint(1, 70)]))
            # the plain form multiplies every expert with as many rows as the fullest one has
            if case["experts"] * m * k <= MAX_WEIGHTS and 2 * m * k * case["experts"] * max(_counts(case)) <= MAX_FLOPS:
                return case
        elif m * k <= MAX_WEIGHTS and 2 * m * case["n"] * k <= MAX_FLOPS:
            return case


def _counts(case):
    """Tokens of every expert: each goes to one of them, popular ones get more and some may get none."""
    rng = random.Random(case["routing"])
    weights = [rng.random() ** 2 + 0.02 for _ in range(case["experts"])]
    counts = [0] * case["experts"]
    for e in rng.choices(range(case["experts"]), weights, k=case["n"]):
        counts[e] += 1
    return counts


def work(case):
    """Activations, the codes and scales of the weights that have tokens, and outputs once each; two operations per product."""
    n, k = case["n"], case["k"]
    if case["op"] == "quantize":  # read once, codes and scales written, numbers written
        return {"bytes": n * k * (BYTES[case["x"]] + BYTES["mx"] + BYTES[case["o"]]), "flops": 0}
    m = case["m"]
    matrices = sum(c > 0 for c in _counts(case)) if case["op"] == "grouped" else 1
    return {"bytes": matrices * m * k * BYTES["mx"] + n * k * BYTES[case["x"]] + n * m * BYTES[case["o"]], "flops": 2 * m * n * k}


# ---- the format, in 32 bits

def _scale_exponents(blocks):
    """Exponent of each block's scale: that of the largest magnitude, less 2 (the exponent of 4, the largest power of two of e2m1)."""
    return (torch.frexp(blocks.abs().amax(-1)).exponent - 1 - 2).clamp(-127, 127)


def _power_of_two(e, dtype):
    return torch.ldexp(torch.ones_like(e, dtype=dtype), e)


def _round_e2m1(a):
    """|numbers| to the nearest of e2m1, ties to the even code: steps of 0.5 up to 2, of 1 up to 4, of 2 up to 6."""
    a = a.clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    return torch.round(a / step) * step


def _fake_quantize(x):
    """The numbers that `x` [..., k] becomes, in 32 bits."""
    blocks = x.float().unflatten(-1, (-1, 32))
    scale = _power_of_two(_scale_exponents(blocks), torch.float32).unsqueeze(-1)
    y = blocks / scale
    return (torch.copysign(_round_e2m1(y.abs()), y) * scale).flatten(-2)


def _pack(x):
    """Codes and scales of `x` [..., rows, k] in the package's layout."""
    k = x.shape[-1]
    blocks = x.float().unflatten(-1, (-1, 32))
    e = _scale_exponents(blocks)
    y = blocks / _power_of_two(e, torch.float32).unsqueeze(-1)
    twice = (_round_e2m1(y.abs()) * 2).to(torch.uint8)  # 0 1 2 3 4 6 8 12
    codes = torch.where(twice <= 4, twice, 5 + (twice >= 8).to(torch.uint8) + (twice >= 12).to(torch.uint8)) | (torch.signbit(y).to(torch.uint8) << 3)
    codes = torch.nn.functional.pad(codes.flatten(-2), (0, -k % 256))
    q = (codes[..., 0::2] | (codes[..., 1::2] << 4)).unflatten(-1, (-1, 128)).transpose(-3, -2).contiguous()
    s = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -(k // 32) % 4)).unflatten(-1, (-1, 4)).transpose(-3, -2).contiguous()
    return q, s


def _numbers(q, s, k, table):
    """The numbers of packed codes [..., rows, k], in the type of `table` (the sixteen numbers of e2m1)."""
    rows = q.transpose(-3, -2).flatten(-2)
    v = table[torch.stack((rows & 15, rows >> 4), -1).int()].flatten(-2)[..., :k]
    e = s.transpose(-3, -2).flatten(-2)[..., :k // 32].int() - 127
    return (v.unflatten(-1, (-1, 32)) * _power_of_two(e, table.dtype).unsqueeze(-1)).flatten(-2)


def _table(dtype, device):
    t = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=dtype, device=device)
    return torch.cat((t, -t))


# ---- what a program has in hand

def _activations(gen, case, rows):
    x = torch.randn((rows, case["k"]), generator=gen, device="cuda")
    heavy = torch.randint(0, case["k"], (max(1, case["k"] // 500),), generator=gen, device="cuda")
    x[:, heavy] *= 20
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n, k, op = case["n"], case["k"], case["op"]
    state = {"case": case}
    if op == "quantize":
        x = torch.randn((n, k), generator=gen, device="cuda").mul_(k ** -0.5) if n > 2048 else _activations(gen, case, n)
        state["x"] = x.to(TYPES[case["x"]])
        state["o"] = torch.empty((n, k), device="cuda", dtype=TYPES[case["o"]])
        return state
    m = case["m"]
    rows = n
    if op == "grouped":
        counts = _counts(case)
        rows = n + case["behind"]
        state["counts"] = counts  # the plain form's batch; the kernels read `offsets`
        state["offsets"] = torch.tensor([sum(counts[:e]) for e in range(len(counts) + 1)], dtype=torch.int32).to("cuda")
        parts = [_pack(torch.randn((m, k), generator=gen, device="cuda").mul_(k ** -0.5)) for _ in counts]
        state["q"], state["s"] = (torch.stack([p[i] for p in parts]) for i in (0, 1))
    else:
        state["q"], state["s"] = _pack(torch.randn((m, k), generator=gen, device="cuda").mul_(k ** -0.5))
    x = _activations(gen, case, rows)
    state["x"], state["xs"] = _pack(x) if case["x"] == "mx" else (x.to(TYPES[case["x"]]), None)
    state["o"] = torch.zeros((rows, m), device="cuda", dtype=TYPES[case["o"]])
    return state


# ---- one pass

def run(state):
    case = state["case"]
    op, k, o = case["op"], case["k"], state["o"]
    if own:
        import tuna_b200

        if op == "quantize":
            q, s = tuna_b200.mx_quantize(state["x"])
            tuna_b200.mx_dequant(q, s, o, case["n"], k)
        elif op == "matmul":
            tuna_b200.mx_matmul(state["x"], state["xs"], state["q"], state["s"], o, case["m"], case["n"], k)
        else:
            tuna_b200.mx_matmul_grouped(state["x"], state["xs"], state["q"], state["s"], state["offsets"], o, case["m"], o.shape[0], k)
        return o
    if op == "quantize":
        return _fake_quantize(state["x"]).to(o.dtype)
    table = _table(torch.float32, o.device)
    x = _fake_quantize(state["x"]) if state["xs"] is None else _numbers(state["x"], state["xs"], k, table)
    w = _numbers(state["q"], state["s"], k, table)
    if op == "matmul":
        return (x @ w.transpose(0, 1)).to(o.dtype)
    # every expert's rows of x, as many for each as the fullest one has, and the rows that are its own back
    most, first = max(state["counts"]), state["offsets"]
    row = first[:-1, None] + torch.arange(most, device=x.device)
    mine = row < first[1:, None]
    y = torch.bmm(x[row.clamp(max=x.shape[0] - 1)], w.transpose(1, 2))
    out = torch.zeros((x.shape[0] + 1, case["m"]), dtype=torch.float32, device=x.device)
    out[torch.where(mine, row, x.shape[0])] = y
    return out[:-1].to(o.dtype)


# ---- the definition in 64 bits

def _two_to(e):
    """2^e in 64 bits, of whole numbers from -127 on (below, a scale cannot go)."""
    return ((e.long().clamp(min=-127) + 1023) << 52).view(torch.float64)


def _exact_numbers(x):
    """Each number of a block goes to the nearest of e2m1 times the block's scale: by the borders between neighbours, the
    border itself to the neighbour with an even code."""
    v = x.double().reshape(*x.shape[:-1], -1, 32)
    largest = v.abs().max(dim=-1, keepdim=True).values
    scale = _two_to((largest.view(torch.int64) >> 52) - 1023 - 2)  # from the bits of the double: its exponent, less 2
    y = v.abs() / scale
    index = torch.zeros_like(y)
    for border, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        index += (y >= border) if up else (y > border)
    magnitude = torch.where(index < 4, index / 2, torch.where(index < 6, index - 2, 2 * index - 8))
    return (torch.sign(v) * magnitude * scale).reshape(x.shape)


def _exact_decoded(q, s, k):
    """A matrix's numbers from the bits of its codes (sign, two of exponent, one of mantissa) and scales."""
    out = torch.empty((q.shape[1], 256 * q.shape[0]), dtype=torch.float64, device=q.device)
    for odd in (0, 1):
        c = (q >> 4 * odd) & 15
        exponent, mantissa = ((c >> 1) & 3).double(), (c & 1).double()
        v = torch.where(exponent > 0, torch.exp2(exponent - 1) * (1 + mantissa / 2), mantissa / 2)
        out[:, odd::2] = torch.where(c >= 8, -v, v).permute(1, 0, 2).reshape(q.shape[1], -1)
    scale = _two_to(s.long() - 127).permute(1, 0, 2).reshape(s.shape[1], -1)[:, :k // 32]
    return out[:, :k] * scale.repeat_interleave(32, 1)


def exact(case, seed):
    state = prepare(case, seed)
    k = case["k"]
    if case["op"] == "quantize":
        return _exact_numbers(state["x"])
    x = _exact_numbers(state["x"]) if state["xs"] is None else _exact_decoded(state["x"], state["xs"], k)
    if case["op"] == "matmul":
        return torch.einsum("nk,mk->nm", x, _exact_decoded(state["q"], state["s"], k))
    out = torch.zeros(state["o"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for e, count in enumerate(state["counts"]):
        if count:
            out[first:first + count] = torch.einsum("nk,mk->nm", x[first:first + count], _exact_decoded(state["q"][e], state["s"][e], k))
        first += count
    return out
