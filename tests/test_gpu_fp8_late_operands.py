"""Every operand of the 8-bit gradients written by the kernel right before the call, which lets its dependents start before it writes: a slice of the operand at its end, so that large ones, those of
the forms that only large calls take, are tested as small ones are."""

import pytest
import torch

import tuna_b200
from tests.gpu_util import stream_ptr
from tests.test_gpu_mx_stream_order import LATE_WRITER
from tuna_b200 import _lib

pytestmark = pytest.mark.gpu
SLICE = 64 << 10  # bytes that come late: what the slow writer does in a fraction of a millisecond


def finish():
    torch.cuda.synchronize()
    assert _lib.load().tuna_check_device_status(stream_ptr()) == 0


def late_slice(name, args, call, outputs, graph):
    call(args)
    finish()
    want = [o.clone() for o in outputs]
    assert all(torch.isfinite(w).all() and float(w.float().std()) > 1e-4 for w in want)
    right = args[name].view(torch.uint8).flatten()
    late = right.clone()
    end = late[-SLICE:]
    end.zero_()
    # without the slice the results are others
    call({**args, name: late.view(args[name].dtype).view(args[name].shape)})
    finish()
    assert not all(torch.equal(o, w) for o, w in zip(outputs, want))
    writer = torch.cuda._compile_kernel(LATE_WRITER, "late_writer")
    pair = [end, right[-SLICE:], end.numel()]

    def calls():
        writer(grid=(1, 1, 1), block=(256, 1, 1), args=pair + pair)
        call({**args, name: late.view(args[name].dtype).view(args[name].shape)})

    run = calls
    if graph:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                calls()
        run = g.replay
    for _ in range(3):
        end.zero_()
        for o in outputs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        run()
        finish()
        assert all(torch.equal(o, w) for o, w in zip(outputs, want))


# features (the products have twice as many), tokens, columns.  Gradients in one launch, dw beside dx (above 2^35 products), z and dh streamed (at least 296 tiles of 128 x 128)
SIZES = [(144, 300, 272), (2048, 2500, 48), (4096, 1200, 4096)]


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("name", ["x", "xs", "q", "s", "dy"])
@pytest.mark.parametrize("f,n,k", SIZES)
def test_operands_of_a_products_gradients(f, n, k, name, graph):
    check(f, n, k, name, graph, False)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("name", ["x", "xs", "q", "s", "dy", "z"])
@pytest.mark.parametrize("f,n,k", SIZES)
def test_operands_of_a_gated_blocks_gradients(f, n, k, name, graph):
    check(f, n, k, name, graph, True)


def check(f, n, k, name, graph, gated):
    gen = torch.Generator(device="cuda").manual_seed(n)
    q, s = tuna_b200.fp8_quantize(torch.randn(2 * f, k, generator=gen, device="cuda"), "square")
    x = torch.randn(n, k, generator=gen, device="cuda", dtype=torch.bfloat16)
    codes = name == "xs" or (name == "x" and graph)  # x in 16 bits, and as codes
    args = {**(dict(zip(("x", "xs"), tuna_b200.fp8_quantize(x, "column"))) if codes else {"x": x}), "q": q, "s": s}
    args["dy"] = torch.randn(n, f if gated else 2 * f, generator=gen, device="cuda", dtype=torch.bfloat16)
    if gated:
        args["z"] = torch.randn(n, 2 * f, generator=gen, device="cuda", dtype=torch.bfloat16)
    dx, dw = torch.empty(n, k, device="cuda"), torch.empty(2 * f, k, device="cuda")

    def call(a):
        if gated:
            tuna_b200.fp8_gated_backward(a["dy"], a["z"], a["x"], a.get("xs"), a["q"], a["s"], dx, dw, f, n, k)
        else:
            tuna_b200.fp8_matmul_backward(a["dy"], a["x"], a.get("xs"), a["q"], a["s"], dx, dw, 2 * f, n, k)

    late_slice(name, args, call, [dx, dw], graph)
