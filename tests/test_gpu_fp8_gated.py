"""The gated block of 8-bit block-scaled matrices and its gradients on the GPU, against 64 bits with the bounds that fp8_util derives."""

import math

import numpy as np
import pytest
import torch

import tuna_b200
from oracle import fp8_oracle as fo
from tests.fp8_util import STEP32, check, check_product, gated, gated_gradient, numpy64, quantized_range, random_matrix, rounded, sums
from tests.gpu_util import Guarded
from tuna_b200 import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
KINDS = ["silu", "gelu"]


def finish():
    torch.cuda.synchronize()
    assert _lib.load().tuna_check_device_status(torch.cuda.current_stream().cuda_stream) == 0


def guarded(rows, cols, dtype):
    hold = Guarded(rows * cols * dtype.itemsize, dtype, (rows, cols))
    hold.view.fill_(float("nan"))
    return hold


def weights(f, k, seed):
    """A matrix [2f, k] whose projections are of the size that they have in a model: a few units."""
    (q, s), w = random_matrix(2 * f, k, "square", seed, spread=1)
    s -= int(np.round(np.log2(40 * np.sqrt(k))))
    w = w * 2.0 ** -int(np.round(np.log2(40 * np.sqrt(k))))
    return (q, s), w


def forward(f, n, k, dtype=torch.float32, kind="silu", seed=0, with_z=False, codes=False):
    (q, s), w = weights(f, k, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, k, generator=gen, device="cuda").to(torch.bfloat16 if dtype == torch.float32 else dtype)
    h = guarded(n, f, dtype)
    z = guarded(n, 2 * f, dtype) if with_z else None
    given = tuna_b200.fp8_quantize(x) if codes else (x, None)
    tuna_b200.fp8_gated(*given, q, s, h.view, f, n, k, kind, z=z.view if z else None)
    finish()
    assert h.guards_intact()
    ref_z, z_off, ref_h, h_off = gated(fo.numbers(numpy64(x), "row"), w, kind)
    check(h.view, ref_h, rounded(ref_h, h_off, dtype))
    if z:
        assert z.guards_intact()
        check(z.view, ref_z, rounded(ref_z, z_off, dtype))
    return x, (q, s), w, h.view, z.view if z else None


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("f,n,k", [(16, 1, 16), (128, 1, 4096), (1360, 3, 784), (4096, 16, 400), (64, 17, 272), (144, 43, 1040), (1008, 130, 528), (256, 300, 144), (720, 700, 272)])
def test_gated(f, n, k, dtype, kind):
    forward(f, n, k, dtype, kind, seed=f + n, with_z=dtype != torch.float32)


@pytest.mark.parametrize("n", [1, 2, 8, 9, 15, 16, 17, 31, 33, 64, 65, 127, 129, 193, 240, 257, 400, 513])
def test_tokens(n):
    forward(272, n, 272, torch.bfloat16, seed=n, with_z=n % 2 == 1, codes=n % 3 == 0)


@pytest.mark.parametrize("f", [16, 48, 144, 592, 1184, 2368, 4736, 9472, 14336])
@pytest.mark.parametrize("n", [1, 9])
def test_row_tiles_of_every_height(f, n):
    forward(f, n, 400, torch.float16, seed=f, with_z=n == 9)
    forward(f, n, 144, torch.float32, "gelu", seed=f, codes=True)


def test_z_changes_nothing_else():
    f, n, k = 400, 50, 272
    x, w, _, h, z = forward(f, n, k, torch.bfloat16, with_z=True)
    other = torch.empty_like(h)
    tuna_b200.fp8_gated(x, None, *w, other, f, n, k)
    both = torch.empty(n, 2 * f, device="cuda", dtype=torch.bfloat16)
    tuna_b200.fp8_matmul(x, None, *w, both, 2 * f, n, k)
    finish()
    assert torch.equal(h, other) and torch.equal(z, both)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [3, 40])
def test_large_and_infinite_projections(n, kind):
    """Gates of any size: nothing overflows that the formula does not, and what is no number stays in its row."""
    f, k = 128, 128
    x = torch.zeros(n, k, device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 1
    w = torch.zeros(2 * f, k)
    w[:f, 0] = torch.cat((torch.linspace(-300, 300, f - 28), torch.tensor([-1e30, 1e30, -3e4, 3e4] * 7)))
    w[f:, 0] = 0.5
    q, s = tuna_b200.fp8_quantize(w.cuda(), "square")
    h = torch.empty(n, f, device="cuda")
    tuna_b200.fp8_gated(x, None, q, s, h, f, n, k, kind)
    finish()
    o = torch.empty(2 * f, k, device="cuda")
    tuna_b200.fp8_dequant(q, s, o, 2 * f, k)
    with np.errstate(over="ignore", invalid="ignore"):
        _, _, ref, off = gated(fo.numbers(numpy64(x), "row"), numpy64(o), kind)
    check(h, ref, rounded(ref, off, torch.float32))
    x[1, 5] = float("nan")
    tuna_b200.fp8_gated(x, None, q, s, h, f, n, k, kind)
    finish()
    assert torch.isnan(h[1]).all() and not torch.isnan(h[0]).any() and not torch.isnan(h[2:]).any()


def backward(f, n, k, kind="silu", seed=0, dtype=torch.bfloat16, dx_type=torch.float32, dw_type=torch.float32, codes=False):
    (q, s), w = weights(f, k, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, k, generator=gen, device="cuda").to(dtype)
    z = (torch.randn(n, 2 * f, generator=gen, device="cuda") * 2).to(dtype)
    dh = torch.randn(n, f, generator=gen, device="cuda").to(dtype)
    dh[n - n // 8:] = 0
    dx, dw = guarded(n, k, dx_type), guarded(2 * f, k, dw_type)
    given = tuna_b200.fp8_quantize(x, "column") if codes else (x, None)
    tuna_b200.fp8_gated_backward(dh, z, *given, q, s, dx.view, dw.view, f, n, k, kind)
    finish()
    assert dx.guards_intact() and dw.guards_intact()
    dy, off = gated_gradient(numpy64(dh), numpy64(z), kind)
    a, a_off = quantized_range(dy, off, "row")
    ref, sum_off = sums(a, w, a_off)
    check(dx.view, ref, rounded(ref, sum_off, dx_type))
    b, b_off = quantized_range(dy, off, "column")
    ref, sum_off = sums(b.T, fo.numbers(numpy64(x), "column"), b_off.T)
    check(dw.view, ref, rounded(ref, sum_off, dw_type))
    return dh, z, x, (q, s), dx.view, dw.view


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("f,n,k", [(16, 1, 16), (128, 128, 128), (64, 3, 272), (144, 129, 144), (272, 17, 1040), (720, 301, 528), (1360, 333, 784), (48, 1030, 96), (2304, 40, 48)])
def test_gradients(f, n, k, kind):
    backward(f, n, k, kind, seed=f + n)


@pytest.mark.parametrize("f,n,kind,dtype", [(2048, 2500, "silu", torch.bfloat16), (12800, 385, "gelu", torch.float16)])
def test_gradients_of_many_tiles(f, n, kind, dtype):
    """As many as stream through: more than two of 128 x 128 for every SM, and rows that end inside one."""
    backward(f, n, 16, kind, seed=n, dtype=dtype)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("f,n", [(2048, 2500), (256, 300), (144, 300)])
def test_gradients_that_are_no_numbers_spoil_their_own_blocks(f, n, bad):
    """Of dx the rows of tokens, of dw the rows of features, that have one."""
    k = 16
    (q, s), _ = weights(f, k, 3)
    x, z, dh = (torch.randn(n, c, device="cuda", dtype=torch.bfloat16) for c in (k, 2 * f, f))
    dh[7, 3] = dh[n - 1, f - 1] = bad
    dx, dw = torch.empty(n, k, device="cuda"), torch.empty(2 * f, k, device="cuda")
    tuna_b200.fp8_gated_backward(dh, z, x, None, q, s, dx, dw, f, n, k)
    finish()
    rows = torch.zeros(n, dtype=torch.bool, device="cuda")
    rows[[7, n - 1]] = True
    assert torch.equal(torch.isnan(dx), rows[:, None].expand(n, k))
    rows = torch.zeros(2 * f, dtype=torch.bool, device="cuda")
    rows[[3, f - 1, f + 3, 2 * f - 1]] = True
    assert torch.equal(torch.isnan(dw), rows[:, None].expand(2 * f, k))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("f,n", [(144, 300), (256, 300), (2048, 2500)])
def test_the_gradient_is_that_of_elementary_operations_in_32_bits(f, n, dtype, kind):
    """Bit for bit, before it is quantized: so its codes are those of the same formula written with torch, in every form of the quantizer."""
    gen = torch.Generator(device="cuda").manual_seed(f)
    z = (torch.randn(n, 2 * f, generator=gen, device="cuda") * 3).to(dtype)
    z[0, :f] = torch.linspace(-200, 200, f).to(dtype)
    dh = torch.randn(n, f, generator=gen, device="cuda").to(dtype)
    k = -(-n // 16) * 16
    x = torch.eye(n, k, device="cuda", dtype=dtype)  # picks the numbers one by one
    dw = torch.empty(2 * f, k, device="cuda")
    tuna_b200.fp8_gated_backward(dh, z, x, None, None, None, None, dw, f, n, k, kind)
    finish()
    g, u = z.float().split(f, 1)
    p, slope = g, torch.ones_like(g)
    if kind == "gelu":
        c = 2 * math.sqrt(2 / math.pi)
        p, slope = c * (g + 0.044715 * (g * g * g)), c * (1 + 3 * 0.044715 * (g * g))
    sigma = 1 / (1 + torch.exp(-p))
    d = dh.float()
    dy = torch.cat((d * u * (sigma + g * sigma * (1 - sigma) * slope), d * g * sigma), 1)
    q, s = tuna_b200.fp8_quantize(dy, "column")
    want = torch.empty(n, 2 * f, device="cuda")
    tuna_b200.fp8_dequant(q, s, want, n, 2 * f, "column")
    assert torch.equal(dw[:, :n].T, want)


@pytest.mark.parametrize("types", [(torch.float16, torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32, torch.float16)], ids=str)
@pytest.mark.parametrize("codes", [False, True])
def test_types_of_the_gradients(types, codes):
    backward(208, 200, 400, "gelu", 1, *types, codes=codes)


def test_either_gradient_alone_is_the_same():
    f, n, k = 208, 333, 272
    dh, z, x, w, dx, dw = backward(f, n, k, seed=4)
    one, other = torch.empty_like(dx), torch.empty_like(dw)
    tuna_b200.fp8_gated_backward(dh, z, None, None, *w, one, None, f, n, k)
    tuna_b200.fp8_gated_backward(dh, z, x, None, None, None, None, other, f, n, k)
    finish()
    assert torch.equal(one, dx) and torch.equal(other, dw)


@pytest.mark.parametrize("kind", KINDS)
def test_gradients_against_differences(kind):
    """Central differences of the block itself: x moves by eighths, which its codes hold.  What the difference may be off from the gradient's
    product with the step: the third derivative's term, the fp32 of h over the step, and the gradient's own rounding, half a step of e4m3 of
    each entry of dy (2^-4 relative; entries far below their block's largest, half of the smallest step)."""
    f, n, k = 144, 20, 128
    rng = np.random.default_rng(1)
    x = rng.integers(-7, 8, (n, k)) / 4
    v = rng.choice([-1.0, 1.0], (n, k)) * (rng.random((n, k)) < 0.05)
    (q, s), w = weights(f, k, 3)
    dh = rng.standard_normal((n, f))
    dh = numpy64(torch.from_numpy(dh).bfloat16())
    step = 0.125

    def value(x):
        t = torch.from_numpy(x).cuda().bfloat16()
        h, z = torch.empty(n, f, device="cuda"), torch.empty(n, 2 * f, device="cuda", dtype=torch.bfloat16)
        tuna_b200.fp8_gated(t, None, q, s, h, f, n, k, kind)
        return numpy64(h)

    def exact(x):
        z = x @ w.T
        return z, fo.activation(z[:, :f], kind)[0] * z[:, f:]

    slope = (value(x + step * v) - value(x - step * v)) / (2 * step)
    z = torch.from_numpy(x @ w.T).cuda().bfloat16()
    dx = torch.empty(n, k, device="cuda")
    tuna_b200.fp8_gated_backward(torch.from_numpy(dh).cuda().bfloat16(), z, None, None, q, s, dx, None, f, n, k, kind)
    finish()
    z64 = numpy64(z)
    dy, off = gated_gradient(dh, z64, kind)
    scale = np.ldexp(1.0, fo.spread(fo.scale_of(fo.largest(np.abs(dy), "row")), "row", n, 2 * f))
    dy_off = off + np.maximum(np.abs(dy) * 2.0 ** -4, scale * 2.0 ** -10)
    # z was rounded for the gradient: half a step of bf16 of each, times the second derivatives (below 1 of the activation, times u, or once)
    z_off = np.abs(x @ w.T) * 2.0 ** -8
    g_off, u_off, u = z_off[:, :f], z_off[:, f:], np.abs(z64[:, f:])
    dy_off = dy_off + np.concatenate((np.abs(dh) * (1.13 * u_off + (u + u_off) * g_off), np.abs(dh) * 1.13 * g_off), 1)
    moved = v @ w.T
    mg, mu = np.abs(moved[:, :f]), np.abs(moved[:, f:])
    # third derivative of a(g) u along the step: a''' u mg^3 + 3 a'' mu mg^2, |a''| < 1.2, |a'''| < 2
    third = step ** 2 / 6 * (2 * (u + step * mu) * mg ** 3 + 3 * 1.2 * mu * mg ** 2)
    _, h = exact(x)
    _, _, _, h_off = gated(x, w, kind)
    allowed = (np.abs(dh) * (third + 2 * (h_off + 2 * STEP32 * np.abs(h)) / step)).sum(1) + (dy_off * np.abs(moved)).sum(1)
    want = (dh * slope).sum(1)
    got = (numpy64(dx) * v).sum(1)
    assert (np.abs(got - want) <= allowed).all()
    assert np.corrcoef(got, want)[0, 1] > 0.99  # and the bound is not what makes it pass


def test_a_padded_batch():
    """Tokens whose gradient is zero take no part, whatever their activations are."""
    f, n, k = 144, 200, 272
    (q, s), w = weights(f, k, 3)
    x = torch.randn(n, k, device="cuda", dtype=torch.bfloat16)
    z = torch.randn(n, 2 * f, device="cuda", dtype=torch.bfloat16)
    dh = torch.randn(n, f, device="cuda", dtype=torch.bfloat16)
    dh[150:] = 0
    out = []
    for rows in (n, 150):
        dx, dw = torch.empty(rows, k, device="cuda"), torch.empty(2 * f, k, device="cuda")
        tuna_b200.fp8_gated_backward(dh[:rows], z[:rows], x[:rows], None, q, s, dx, dw, f, rows, k)
        out.append((dx, dw))
    finish()
    assert torch.equal(out[0][0][:150], out[1][0]) and not out[0][0][150:].any()
    # x's blocks of a column hold the padding's activations: these numbers differ by their scales only
    a = fo.numbers(numpy64(x), "column")
    dy, off = gated_gradient(numpy64(dh), numpy64(z), "silu")
    b, b_off = quantized_range(dy, off, "column")
    ref, sum_off = sums(b.T, a, b_off.T)
    check(out[0][1], ref, rounded(ref, sum_off, torch.float32))


@pytest.mark.parametrize("n", [1, 2, 16, 100])
def test_a_training_step_of_an_mlp(n):
    """Gated block, down projection and the gradients of both, call after call as a program makes them, captured and replayed."""
    f, k = 272, 400
    up, w_up = weights(f, k, 1)
    down, w_down = random_matrix(k, f, "square", 2, spread=1)
    x = torch.empty(n, k, device="cuda", dtype=torch.bfloat16)
    dy = torch.empty(n, k, device="cuda", dtype=torch.bfloat16)
    h, dh = (torch.empty(n, f, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    z = torch.empty(n, 2 * f, device="cuda", dtype=torch.bfloat16)
    y, dx = torch.empty(n, k, device="cuda"), torch.empty(n, k, device="cuda")
    dw_up, dw_down = torch.empty(2 * f, k, device="cuda"), torch.empty(k, f, device="cuda")

    def step():
        tuna_b200.fp8_gated(x, None, *up, h, f, n, k, z=z)
        tuna_b200.fp8_matmul(h, None, *down, y, k, n, f)
        tuna_b200.fp8_matmul_backward(dy, h, None, *down, dh, dw_down, k, n, f)
        tuna_b200.fp8_gated_backward(dh, z, x, None, *up, dx, dw_up, f, n, k)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(2):
        x.copy_(torch.randn(n, k, device="cuda"))
        dy.copy_(torch.randn(n, k, device="cuda"))
        graph.replay()
        finish()
        results = [t.clone() for t in (h, z, y, dh, dx, dw_up, dw_down)]
        step()
        finish()
        assert all(torch.equal(a, b) for a, b in zip(results, (h, z, y, dh, dx, dw_up, dw_down)))
    x64, dy64, h64, dh64 = (numpy64(t) for t in (x, dy, h, dh))
    ref_z, z_off, ref_h, h_off = gated(fo.numbers(x64, "row"), w_up, "silu")
    check(z, ref_z, rounded(ref_z, z_off, z.dtype))
    check(h, ref_h, rounded(ref_h, h_off, h.dtype))
    check_product(y, fo.numbers(h64, "row"), w_down.T)
    check_product(dh, fo.numbers(dy64, "row"), w_down)
    check_product(dw_down, fo.numbers(dy64, "column").T, fo.numbers(h64, "column"))
    g, off = gated_gradient(dh64, numpy64(z), "silu")
    a, a_off = quantized_range(g, off, "row")
    ref, sum_off = sums(a, w_up, a_off)
    check(dx, ref, rounded(ref, sum_off, dx.dtype))
    b, b_off = quantized_range(g, off, "column")
    ref, sum_off = sums(b.T, fo.numbers(x64, "column"), b_off.T)
    check(dw_up, ref, rounded(ref, sum_off, dw_up.dtype))


def test_refusals():
    f, n, k = 32, 4, 64
    (q, s), _ = weights(f, k, 1)
    x, h = torch.zeros(n, k, device="cuda", dtype=torch.float16), torch.zeros(n, f, device="cuda", dtype=torch.float16)
    z = torch.zeros(n, 2 * f, device="cuda", dtype=torch.float16)
    tuna_b200.fp8_gated(x, None, q, s, h, f, n, k, z=z)
    for kw in ({"z": z.bfloat16()}, {"z": z[:, :f]}, {"z": z.t()}, {"activation": "tanh"}):
        with pytest.raises((TypeError, ValueError)):
            tuna_b200.fp8_gated(x, None, q, s, h, f, n, k, **kw)
    with pytest.raises((TypeError, ValueError)):
        tuna_b200.fp8_gated(x, None, q, s, h.float(), f, n, k, z=z.float())
    with pytest.raises((TypeError, ValueError)):
        tuna_b200.fp8_gated(x, None, q[:f], s, h, f, n, k)
    dx, dw = torch.zeros(n, k, device="cuda"), torch.zeros(2 * f, k, device="cuda")
    tuna_b200.fp8_gated_backward(h, z, x, None, q, s, dx, dw, f, n, k)
    for args in ((h, z.bfloat16(), x, None, q, s, dx, dw), (h, None, x, None, q, s, dx, dw), (h, z, x, None, q, s, None, None), (h, z[:, :f], x, None, q, s, dx, dw), (h, z, x, None, q, s, dx, dw[:f])):
        with pytest.raises((TypeError, ValueError)):
            tuna_b200.fp8_gated_backward(*args, f, n, k)
