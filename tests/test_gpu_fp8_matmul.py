"""Products of 8-bit block-scaled matrices and their gradients on the GPU against sums in 64 bits, with the bounds that fp8_util derives."""

import numpy as np
import pytest
import torch

import tuna_b200
from oracle import fp8_oracle as fo
from tests.fp8_util import check_product, codes_tensor, numpy64, random_matrix
from tests.gpu_util import Guarded
from tuna_b200 import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def finish():
    torch.cuda.synchronize()
    assert _lib.load().tuna_check_device_status(torch.cuda.current_stream().cuda_stream) == 0


def guarded(rows, cols, dtype):
    return Guarded(rows * cols * dtype.itemsize, dtype, (rows, cols))


def product(m, n, k, seed=0, dtype=torch.float32, spread=3):
    (xq, xs), x = random_matrix(n, k, "row", 2 * seed + 1, spread)
    (wq, ws), w = random_matrix(m, k, "square", 2 * seed + 2, spread)
    hold = guarded(n, m, dtype)
    tuna_b200.fp8_matmul(xq, xs, wq, ws, hold.view, m, n, k)
    finish()
    assert hold.guards_intact()
    check_product(hold.view, x, w.T)


def gradients(m, n, k, seed=0, dx_type=torch.float32, dw_type=torch.float32, dy_type=torch.bfloat16, codes=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dy = (torch.randn(n, m, generator=gen, device="cuda") * torch.exp(2 * torch.randn(n, 1, generator=gen, device="cuda"))).to(dy_type)
    x = torch.randn(n, k, generator=gen, device="cuda").to(dy_type)
    x[:, k // 3] *= 40
    (wq, ws), w = random_matrix(m, k, "square", seed)
    dx, dw = guarded(n, k, dx_type), guarded(m, k, dw_type)
    given = tuna_b200.fp8_quantize(x, "column") if codes else (x, None)
    tuna_b200.fp8_matmul_backward(dy, *given, wq, ws, dx.view, dw.view, m, n, k)
    finish()
    assert dx.guards_intact() and dw.guards_intact()
    check_product(dx.view, fo.numbers(numpy64(dy), "row"), w)
    check_product(dw.view, fo.numbers(numpy64(dy), "column").T, fo.numbers(numpy64(x), "column"))
    return dy, x, (wq, ws), dx.view, dw.view


@pytest.mark.parametrize("k", [16, 32, 48, 112, 128, 144, 256, 272, 512, 528, 640, 2064, 4096])
@pytest.mark.parametrize("n", [1, 20])
def test_reduction_lengths(n, k):
    product(144, n, k, seed=k)


@pytest.mark.parametrize("m", [16, 112, 128, 144, 240, 272, 1008, 4096])
def test_output_features(m):
    product(m, 3, 544, seed=m)
    product(m, 70, 160, seed=m)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 300, 513])
def test_tokens(n):
    product(272, n, 784, seed=n, dtype=torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(4096, 1, 4096), (1008, 43, 4112), (6144, 256, 1024), (528, 130, 14336), (20000, 16, 512), (2048, 700, 2048), (48, 2000, 96)])
def test_sizes_and_types(m, n, k, dtype):
    product(m, n, k, seed=m + n, dtype=dtype)


@pytest.mark.parametrize("m", [16, 48, 272, 1184, 2368, 4736, 9472, 18944, 19008, 40000])
@pytest.mark.parametrize("n,k", [(1, 400), (9, 1312), (16, 144)])
def test_row_tiles_of_every_height(m, n, k):
    """Up to 16 tokens: 8 to 128 rows a tile, folded four ways, two ways and not, with and without a remainder, of codes and of 16 bits."""
    product(m, n, k, seed=m)
    x = torch.randn(n, k, device="cuda", dtype=torch.float16)
    (wq, ws), w = random_matrix(m, k, "square", 5)
    o = torch.empty(n, m, device="cuda")
    tuna_b200.fp8_matmul(x, None, wq, ws, o, m, n, k)
    finish()
    check_product(o, fo.numbers(numpy64(x), "row"), w.T)


@pytest.mark.parametrize("n", [17, 33, 49, 65, 97, 129, 161, 177, 193, 225, 241, 257, 353, 400, 530, 1030])
def test_token_tiles_of_every_width(n):
    product(2608, n, 320, seed=n)


@pytest.mark.parametrize("m,n,k", [(384, 40, 1040), (384, 4, 1040), (2048, 300, 528)])
def test_single_products_are_exact(m, n, k):
    """One column of x is not zero: the outputs are w's numbers, so no row, column or scale is taken for another."""
    rng = np.random.default_rng(5)
    (wq, ws), w = random_matrix(m, k, "square", 6, spread=8)
    codes = np.zeros((n, k), dtype=np.uint8)
    at = rng.permutation(k)[:n]
    codes[np.arange(n), at] = 56  # 1.0
    scales = rng.integers(120, 135, (n, -(-k // 128)), dtype=np.uint8)
    o = torch.full((n, m), float("nan"), device="cuda")
    tuna_b200.fp8_matmul(codes_tensor(codes), torch.from_numpy(fo.pack(scales, "row")).cuda(), wq, ws, o, m, n, k)
    finish()
    want = w[:, at].T * 2.0 ** (scales[np.arange(n), at // 128].astype(float) - 127)[:, None]
    assert np.array_equal(o.double().cpu().numpy(), want)


@pytest.mark.parametrize("m,n,k", [(400, 300, 1040), (272, 700, 144), (128, 130, 400)])
def test_single_products_of_the_gradients_are_exact(m, n, k):
    """dy has one entry a row (dx: a row of w each) or one row (dw: products of two numbers)."""
    rng = np.random.default_rng(m)
    (wq, ws), w = random_matrix(m, k, "square", 6, spread=8)
    at = rng.integers(0, m, n)
    dy = torch.zeros(n, m)
    dy[torch.arange(n), torch.from_numpy(at)] = torch.from_numpy(2.0 ** rng.integers(-6, 6, n)).float()
    dx = torch.full((n, k), float("nan"), device="cuda")
    tuna_b200.fp8_matmul_backward(dy.cuda().bfloat16(), None, None, wq, ws, dx, None, m, n, k)
    finish()
    assert np.array_equal(numpy64(dx), w[at] * dy.numpy().astype(float)[np.arange(n), at][:, None])
    row = n // 2 + 3
    dy = torch.zeros(n, m)
    dy[row] = torch.from_numpy(rng.integers(-15, 16, m)).float()
    x = torch.from_numpy(rng.integers(-15, 16, (n, k))).float()
    dw = torch.full((m, k), float("nan"), device="cuda")
    tuna_b200.fp8_matmul_backward(dy.cuda().half(), x.cuda().half(), None, None, None, None, dw, m, n, k)
    finish()
    assert torch.equal(dw.cpu(), torch.outer(dy[row], x[row]))


@pytest.mark.parametrize("m,n,k", [(128, 1, 8192), (4096, 7, 4096), (1024, 16, 14336), (1040, 50, 16384), (4096, 600, 4096), (8192, 300, 28672)])
def test_sums_that_24_bits_hold_are_exact(m, n, k):
    """Small whole numbers: every sum is one too, below 2^24, whatever the order.  An accumulator of fewer bits would show."""
    rng = np.random.default_rng(k)
    x = torch.from_numpy(rng.integers(-15, 16, (n, k))).float().cuda()
    w = torch.from_numpy(rng.integers(-15, 16, (m, k))).float().cuda()
    x[:, ::7], w[:, ::7] = 15, 15  # large ones of one sign among them
    o = torch.empty(n, m, device="cuda")
    tuna_b200.fp8_matmul(x.bfloat16(), None, *tuna_b200.fp8_quantize(w, "square"), o, m, n, k)
    finish()
    assert torch.equal(o.double(), x.double() @ w.double().T)


@pytest.mark.parametrize("m,n,k", [(1040, 4096, 528), (4096, 700, 1024), (12288, 2100, 256), (144, 20000, 400)])
def test_gradients_that_24_bits_hold_are_exact(m, n, k):
    rng = np.random.default_rng(k)
    dy, x, w = (torch.from_numpy(rng.integers(-15, 16, s)).float().cuda() for s in ((n, m), (n, k), (m, k)))
    dx, dw = torch.empty(n, k, device="cuda"), torch.empty(m, k, device="cuda")
    tuna_b200.fp8_matmul_backward(dy.half(), x.half(), None, *tuna_b200.fp8_quantize(w, "square"), dx, dw, m, n, k)
    finish()
    assert torch.equal(dx.double(), dy.double() @ w.double())
    assert torch.equal(dw.double(), dy.double().T @ x.double())


def test_gradients_against_differences():
    """The product is linear: with whole numbers, moving x (or a weight) by whole numbers moves the sum of dy * o by what dx (or dw) says, exactly."""
    m, n, k = 272, 150, 400
    rng = np.random.default_rng(3)
    dy, x, w, step_x = (torch.from_numpy(rng.integers(-7, 8, s)).float().cuda() for s in ((n, m), (n, k), (m, k), (n, k)))
    step_w = torch.from_numpy(rng.integers(-7, 8, (m, k))).float().cuda()

    def value(x, w):
        o = torch.empty(n, m, device="cuda")
        tuna_b200.fp8_matmul(x.bfloat16(), None, *tuna_b200.fp8_quantize(w, "square"), o, m, n, k)
        return (o.double() * dy.double()).sum()

    dx, dw = torch.empty(n, k, device="cuda"), torch.empty(m, k, device="cuda")
    tuna_b200.fp8_matmul_backward(dy.bfloat16(), x.bfloat16(), None, *tuna_b200.fp8_quantize(w, "square"), dx, dw, m, n, k)
    assert value(x + step_x, w) - value(x, w) == (dx.double() * step_x.double()).sum()
    assert value(x, w + step_w) - value(x, w) == (dw.double() * step_w.double()).sum()


@pytest.mark.parametrize("m,n,k", [(16, 1, 16), (128, 128, 128), (144, 3, 272), (272, 129, 144), (512, 17, 1040), (1552, 301, 1040), (528, 1025, 784), (2304, 520, 48), (48, 260, 2064)])
def test_gradients(m, n, k):
    gradients(m, n, k, seed=m + n)


@pytest.mark.parametrize("types", [(torch.float16, torch.float32, torch.float16), (torch.bfloat16, torch.bfloat16, torch.bfloat16), (torch.float32, torch.float16, torch.float16)], ids=str)
@pytest.mark.parametrize("codes", [False, True])
def test_types_of_the_gradients(types, codes):
    gradients(272, 200, 400, 1, *types, codes=codes)


def test_either_gradient_alone_is_the_same():
    m, n, k = 400, 333, 272
    dy, x, w, dx, dw = gradients(m, n, k, 5)
    one, other = torch.empty_like(dx), torch.empty_like(dw)
    tuna_b200.fp8_matmul_backward(dy, None, None, *w, one, None, m, n, k)
    tuna_b200.fp8_matmul_backward(dy, x, None, None, None, None, other, m, n, k)
    finish()
    assert torch.equal(one, dx) and torch.equal(other, dw)


def test_a_batch_that_is_padding_gives_zero_gradients():
    m, n, k = 144, 130, 272
    (wq, ws), _ = random_matrix(m, k, "square", 1)
    dx, dw = torch.full((n, k), float("nan"), device="cuda"), torch.full((m, k), float("nan"), device="cuda")
    x = torch.randn(n, k, device="cuda", dtype=torch.float16)
    tuna_b200.fp8_matmul_backward(torch.zeros(n, m, device="cuda", dtype=torch.float16), x, None, wq, ws, dx, dw, m, n, k)
    finish()
    assert not dx.any() and not dw.any()


@pytest.mark.parametrize("n", [5, 20])
def test_scales_of_every_size_and_nan(n):
    """Scales from 2^-50 to 2^50 on either side; a NaN scale or code spoils its own row's or token's outputs and no others."""
    m, k = 256, 1040
    (xq, xs), x = random_matrix(n, k, "row", 1, spread=50)
    (wq, ws), w = random_matrix(m, k, "square", 2, spread=50)

    def run():
        o = torch.empty(n, m, device="cuda")
        tuna_b200.fp8_matmul(xq, xs, wq, ws, o, m, n, k)
        finish()
        check_product(o, x, w.T)

    run()
    xs[1, 3, 2] = 255  # columns 768 .. 895 of token 3
    x[3, 768:896] = np.nan
    run()
    wq.view(torch.uint8)[200, 77] = 0x7f
    w[200, 77] = np.nan
    run()
    ws[0, 8] = 255
    w[:128, 1024:] = np.nan
    run()


@pytest.mark.parametrize("n", [1, 3, 16, 40])
def test_scale_bytes_at_their_ends(n):
    """Bytes 0 and 254, against one another: products of any size that fp32 holds."""
    m, k = 144, 272
    codes = np.full((n, k), 56, dtype=np.uint8)
    low, high = np.zeros((n, 3), dtype=np.uint8), np.full((2, 3), 254, dtype=np.uint8)
    (wq, _), _ = random_matrix(m, k, "square", 3, spread=0)
    w = fo.decode(wq.view(torch.uint8).cpu().numpy(), high, "square")
    o = torch.empty(n, m, device="cuda")
    tuna_b200.fp8_matmul(codes_tensor(codes), torch.from_numpy(fo.pack(low, "row")).cuda(), wq, torch.from_numpy(high).cuda(), o, m, n, k)
    finish()
    check_product(o, fo.decode(codes, low, "row"), w.T)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("m,n,k", [(128, 1, 16), (512, 5, 2064), (1024, 40, 4096), (256, 300, 784), (4096, 2, 14336), (4096, 16, 4096)])
def test_tokens_in_16_bits_are_quantized_by_the_call(m, n, k, dtype):
    x = torch.randn(n, k, device="cuda").to(dtype)
    x[:, 3] *= 30
    (wq, ws), w = random_matrix(m, k, "square", 4)
    o = torch.empty(n, m, device="cuda", dtype=dtype)
    tuna_b200.fp8_matmul(x, None, wq, ws, o, m, n, k)
    finish()
    check_product(o, fo.numbers(numpy64(x), "row"), w.T)
    o2 = torch.empty_like(o)
    tuna_b200.fp8_matmul(*tuna_b200.fp8_quantize(x), wq, ws, o2, m, n, k)
    assert torch.equal(o, o2)


@pytest.mark.parametrize("n", [1, 2, 5, 16, 40])
def test_tokens_with_infinities_and_nan_spoil_only_their_own_outputs(n):
    m, k = 208, 1184
    (wq, ws), w = random_matrix(m, k, "square", 8)
    x = torch.randn(n, k, device="cuda", dtype=torch.bfloat16)
    x[0, 5] = float("inf")
    if n > 1:
        x[n - 1, k - 1] = float("nan")
    o = torch.empty(n, m, device="cuda")
    tuna_b200.fp8_matmul(x, None, wq, ws, o, m, n, k)
    finish()
    assert torch.isnan(o[0]).all() and torch.isnan(o[n - 1]).all()
    check_product(o, fo.numbers(numpy64(x), "row"), w.T)


@pytest.mark.parametrize("n", [3, 24, 200])
def test_runs_agree_bit_for_bit_in_any_workspace(n):
    m, k = 2000, 4096
    (wq, ws), _ = random_matrix(m, k, "square", 2)
    x = torch.randn(n, k, device="cuda", dtype=torch.float16)
    dy = torch.randn(n, m, device="cuda", dtype=torch.float16)
    outs = []
    for fill in (None, 0, 255):
        work = None if fill is None else torch.full((4 << 20,), fill, dtype=torch.uint8, device="cuda")
        o, dx, dw = (torch.full(s, float("nan"), device="cuda") for s in ((n, m), (n, k), (m, k)))
        tuna_b200.fp8_matmul(x, None, wq, ws, o, m, n, k, workspace=work)
        tuna_b200.fp8_matmul_backward(dy, x, None, wq, ws, dx, dw, m, n, k, workspace=work)
        outs.append((o, dx, dw))
    finish()
    assert all(torch.equal(a, b) for other in outs[1:] for a, b in zip(outs[0], other))


def test_an_output_of_more_than_2_31_elements():
    m, n, k = 65536, 33000, 48
    (xq, xs), x = random_matrix(n, k, "row", 1)
    (wq, ws), w = random_matrix(m, k, "square", 2)
    o = torch.empty(n, m, device="cuda", dtype=torch.bfloat16)
    tuna_b200.fp8_matmul(xq, xs, wq, ws, o, m, n, k)
    finish()
    for rows in (slice(0, 3), slice(16000, 16003), slice(n - 300, n)):
        check_product(o[rows], x[rows], w.T)


def test_gradients_of_more_than_2_31_elements():
    """dy has them, and so do dw and dx: sums of few products each."""
    m, n, k = 66000 // 16 * 16, 33000, 16
    dy = torch.zeros(n, m, device="cuda", dtype=torch.bfloat16)
    rows = torch.tensor([0, 127, 128, 16001, n - 1], device="cuda")
    dy[rows] = torch.randint(-15, 16, (5, m), device="cuda").bfloat16()
    x = torch.randint(-15, 16, (n, k), device="cuda").bfloat16()
    w = torch.randint(-15, 16, (m, k), device="cuda").bfloat16()
    dx, dw = torch.full((n, k), 1.0, device="cuda"), torch.full((m, k), 1.0, device="cuda")
    tuna_b200.fp8_matmul_backward(dy, x, None, *tuna_b200.fp8_quantize(w, "square"), dx, dw, m, n, k)
    finish()
    want = torch.zeros(n, k, device="cuda")
    want[rows] = (dy[rows].double() @ w.double()).float()
    assert torch.equal(dx, want)
    assert torch.equal(dw.double(), dy[rows].double().T @ x[rows].double())


# ------------------------------------------------------------------ streams, graphs, devices, views

def test_a_layer_forward_and_backward_captured_and_replayed():
    """Forward pass and gradients of one layer in a graph of a side stream, replayed with other inputs, beside a second one of its kind."""
    m, n, k = 528, 130, 400
    side = torch.cuda.Stream()
    cases = []
    for i in range(2):
        (wq, ws), w = random_matrix(m, k, "square", i)
        x, dy = torch.randn(n, k, device="cuda", dtype=torch.bfloat16), torch.randn(n, m, device="cuda", dtype=torch.bfloat16)
        o, dx, dw = (torch.empty(s, device="cuda") for s in ((n, m), (n, k), (m, k)))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            tuna_b200.fp8_matmul(x, None, wq, ws, o, m, n, k)
            tuna_b200.fp8_matmul_backward(dy, x, None, wq, ws, dx, dw, m, n, k)
        cases.append((graph, x, dy, w, o, dx, dw, wq, ws))  # a graph does not keep what it reads
    for turn in range(3):
        for graph, x, dy, *_ in cases:
            x.copy_(torch.randn(n, k, device="cuda") * 2 ** turn)
            dy.copy_(torch.randn(n, m, device="cuda"))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in cases]
        for (graph, *_), s in zip(cases, streams):
            with torch.cuda.stream(s):
                graph.replay()
        finish()
        for _, x, dy, w, o, dx, dw, *_ in cases:
            check_product(o, fo.numbers(numpy64(x), "row"), w.T)
            check_product(dx, fo.numbers(numpy64(dy), "row"), w)
            check_product(dw, fo.numbers(numpy64(dy), "column").T, fo.numbers(numpy64(x), "column"))


def test_calls_on_two_streams_at_once():
    m, n, k = 2048, 100, 2048
    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = []
    for i in range(2):
        (wq, ws), w = random_matrix(m, k, "square", i)
        cases.append((torch.randn(n, k, device="cuda", dtype=torch.bfloat16), wq, ws, w, torch.empty(n, m, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(10):
        for (x, wq, ws, _, o), s in zip(cases, streams):
            with torch.cuda.stream(s):
                tuna_b200.fp8_matmul(x, None, wq, ws, o, m, n, k)
    finish()
    for x, _, _, w, o in cases:
        check_product(o, fo.numbers(numpy64(x), "row"), w.T)


def test_gradients_on_two_streams_at_once():
    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = []
    for i, (m, n, k) in enumerate([(1040, 300, 528), (4096, 1500, 6144)]):  # dx and dw in one launch, and in two
        gen = torch.Generator(device="cuda").manual_seed(i)
        dy, x, w = (torch.randint(-3, 4, s, generator=gen, device="cuda").float() for s in ((n, m), (n, k), (m, k)))  # whole numbers, sums below 2^24
        cases.append((dy, x, w, dy.half(), x.half(), tuna_b200.fp8_quantize(w, "square"), torch.empty(n, k, device="cuda"), torch.empty(m, k, device="cuda"), (m, n, k)))
    torch.cuda.synchronize()
    for _ in range(10):
        for (_, _, _, dy, x, weights, dx, dw, sizes), s in zip(cases, streams):
            with torch.cuda.stream(s):
                tuna_b200.fp8_matmul_backward(dy, x, None, *weights, dx, dw, *sizes)
    finish()
    for dy, x, w, _, _, _, dx, dw, _ in cases:
        assert torch.equal(dx, dy @ w) and torch.equal(dw, dy.T @ x)


@pytest.mark.parametrize("k", [16, 144, 2064, 2576, 4112])
@pytest.mark.parametrize("n", [1, 5, 16, 40])
@pytest.mark.parametrize("m", [272, 9472, 18944])
def test_what_the_last_scale_word_has_behind_the_last_block_is_not_used(m, n, k):
    (wq, ws), _ = random_matrix(m, k, "square", 1)
    x = torch.randn(n, k, device="cuda", dtype=torch.float16)
    outs = []
    for fill in (0, 255):
        xq, xs = tuna_b200.fp8_quantize(x)
        xs[-1, :, -(-k // 128) % 4 or 4:] = fill
        o = torch.empty(n, m, device="cuda")
        tuna_b200.fp8_matmul(xq, xs, wq, ws, o, m, n, k)
        outs.append(o)
    dy = torch.randn(n, m, device="cuda", dtype=torch.float16)
    for fill in (0, 255):
        xq, xs = tuna_b200.fp8_quantize(x, "column")
        xs[-1, :, -(-n // 128) % 4 or 4:] = fill
        dw = torch.empty(m, k, device="cuda")
        tuna_b200.fp8_matmul_backward(dy, xq, xs, None, None, None, dw, m, n, k)
        outs.append(dw)
    finish()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[2], outs[3])


@pytest.mark.parametrize("n", [4, 90])
def test_a_chain_of_layers_follows_stream_order(n):
    """Every layer's output is the next one's input, without anything in between; small whole numbers, so that the chain is exact."""
    k = 512
    rng = np.random.default_rng(0)
    w = np.zeros((k, k))
    w[np.arange(k), rng.permutation(k)] = 1  # a permutation: numbers move, none changes
    q, s = tuna_b200.fp8_quantize(torch.from_numpy(w).float().cuda(), "square")
    x = torch.from_numpy(rng.integers(-15, 16, (n, k))).cuda().bfloat16()
    a, b = x.clone(), torch.empty_like(x)
    for _ in range(30):
        tuna_b200.fp8_matmul(a, None, q, s, b, k, n, k)
        a, b = b, a
    finish()
    want = numpy64(x)
    for _ in range(30):
        want = want @ w.T
    assert np.array_equal(numpy64(a), want)


def test_row_ranges_are_views():
    """Tokens and, by multiples of 128, weights are taken as views of larger matrices."""
    m, n, k = 512, 64, 400
    (wq, ws), w = random_matrix(m, k, "square", 1)
    x = torch.randn(n, k, device="cuda", dtype=torch.float16)
    o = torch.empty(20, 256, device="cuda")
    tuna_b200.fp8_matmul(x[30:50], None, wq[128:384], ws[1:3], o, 256, 20, k)
    finish()
    check_product(o, fo.numbers(numpy64(x[30:50]), "row"), w[128:384].T)


def test_refusals():
    m, n, k = 32, 4, 64
    (wq, ws), _ = random_matrix(m, k, "square", 1)
    x, o = torch.zeros(n, k, device="cuda", dtype=torch.float16), torch.zeros(n, m, device="cuda")
    xq, xs = tuna_b200.fp8_quantize(x)
    tuna_b200.fp8_matmul(x, None, wq, ws, o, m, n, k)
    for args in ((x, xs, wq, ws, o, m, n, k), (xq, None, wq, ws, o, m, n, k), (x.float(), None, wq, ws, o, m, n, k), (x, None, wq.view(torch.uint8), ws, o, m, n, k),
                 (x, None, wq, ws, o.double(), m, n, k), (x, None, wq, ws, o, m, n + 1, k), (x, None, wq, ws, o.t(), m, n, k), (x, None, wq, ws.cpu(), o, m, n, k),
                 (x, None, wq, None, o, m, n, k), (x, None, wq, ws[:0], o, m, n, k)):
        with pytest.raises((TypeError, ValueError)):
            tuna_b200.fp8_matmul(*args)
    with pytest.raises(tuna_b200.TunaError):
        tuna_b200.fp8_matmul(x[:0], None, wq, ws, o[:0], m, 0, k)
    dy = torch.zeros(n, m, device="cuda", dtype=torch.float16)
    dx, dw = torch.zeros(n, k, device="cuda"), torch.zeros(m, k, device="cuda")
    for args in ((dy, x, None, wq, ws, None, None), (dy.float(), x, None, wq, ws, dx, dw), (dy, x, None, None, None, dx, dw), (dy, None, None, wq, ws, dx, dw),
                 (dy, x, None, wq, ws, dw, dx.t()), (dy, xq, xs, wq, ws, dx, dw), (dy, x, None, wq, ws, dx, dw.cpu())):
        if args[1] is xq:  # scales by row: as many as by column only by chance, here not
            assert xs.numel() != 4 * k
        with pytest.raises((TypeError, ValueError)):
            tuna_b200.fp8_matmul_backward(*args, m, n, k)
    with pytest.raises(tuna_b200.TunaError, match="workspace"):
        tuna_b200.fp8_matmul_backward(dy, x, None, wq, ws, dx, dw, m, n, k, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_tensors_of_a_device_that_is_not_current():
    m, n, k = 144, 20, 272
    (wq, ws), w = random_matrix(m, k, "square", 1)
    x = torch.randn(n, k, dtype=torch.float16)
    o = torch.empty(n, m, device="cuda:1")
    tuna_b200.fp8_matmul(x.to("cuda:1"), None, wq.to("cuda:1"), ws.to("cuda:1"), o, m, n, k)
    torch.cuda.synchronize("cuda:1")
    check_product(o, fo.numbers(numpy64(x), "row"), w.T)
