"""What the 8-bit calls see of the kernels before them in their stream, and the kernels behind of them, without a synchronisation in between."""

import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import tuna_b200
from tests.gpu_util import stream_ptr
from tests.test_gpu_mx_stream_order import LATE_WRITER
from tuna_b200 import _lib

pytestmark = pytest.mark.gpu


def finish():
    torch.cuda.synchronize()
    assert _lib.load().tuna_check_device_status(stream_ptr()) == 0


# ------------------------------------------------------------------ steps of several layers, each reading what the one before wrote

# (features of the block's inside, tokens, width): forms for one token to many, gradients in one launch, beside one another, streamed and not
STEPS = {
    "1": (400, 1, 528),
    "16": (1024, 16, 2048),
    "40": (272, 40, 528),
    "300": (1360, 300, 784),
    "2000": (2560, 2000, 1024),
    "large": (4096, 1300, 4096),
}


class Steps:
    """Forward and backward pass of two MLPs, one behind the other."""

    def __init__(self, f, n, k):
        self.sizes = f, n, k
        gen = torch.Generator(device="cuda").manual_seed(n)
        weight = lambda rows, cols: tuna_b200.fp8_quantize(torch.randn(rows, cols, generator=gen, device="cuda") * cols ** -0.5, "square")  # noqa: E731
        self.up, self.down = [weight(2 * f, k) for _ in range(2)], [weight(k, f) for _ in range(2)]
        new = lambda *shape: torch.empty(shape, device="cuda", dtype=torch.bfloat16)  # noqa: E731
        self.x = [new(n, k) for _ in range(3)]
        self.d = [new(n, k) for _ in range(3)]
        self.h, self.z, self.dh = [new(n, f) for _ in range(2)], [new(n, 2 * f) for _ in range(2)], new(n, f)
        self.dw = [torch.empty(s, device="cuda") for s in ((2 * f, k), (k, f)) for _ in range(2)]
        self.inputs = [(torch.randn(n, k, generator=gen, device="cuda").bfloat16(), torch.randn(n, k, generator=gen, device="cuda").bfloat16()) for _ in range(2)]

    def run(self, between=lambda: None):
        f, n, k = self.sizes
        for i in range(2):
            tuna_b200.fp8_gated(self.x[i], None, *self.up[i], self.h[i], f, n, k, z=self.z[i])
            between()
            tuna_b200.fp8_matmul(self.h[i], None, *self.down[i], self.x[i + 1], k, n, f)
            between()
        for i in (1, 0):
            tuna_b200.fp8_matmul_backward(self.d[i + 1], self.h[i], None, *self.down[i], self.dh, self.dw[2 + i], k, n, f)
            between()
            tuna_b200.fp8_gated_backward(self.dh, self.z[i], self.x[i], None, *self.up[i], self.d[i], self.dw[i], f, n, k)
            between()

    def results(self):
        return [self.x[2], self.d[0], *self.dw]

    def start(self, x, dy):
        for t in (*self.x, *self.d, *self.h, *self.z, self.dh, *self.dw):
            t.fill_(float("nan"))
        self.x[0].copy_(x)
        self.d[2].copy_(dy)


@pytest.mark.parametrize("name", STEPS)
def test_steps_whose_outputs_are_the_next_ones_inputs(name):
    """The same bits as with a synchronisation after every call, eager and replayed, with new inputs every time."""
    steps = Steps(*STEPS[name])
    want = []
    for x, dy in steps.inputs:
        steps.start(x, dy)
        steps.run(torch.cuda.synchronize)
        want.append([t.clone() for t in steps.results()])
        assert all(torch.isfinite(t).all() and float(t.float().std()) > 1e-4 for t in want[-1])
    assert not torch.equal(want[0][1], want[1][1])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        steps.run()
    for run in (steps.run, graph.replay):
        for _ in range(3):
            for (x, dy), w in zip(steps.inputs, want):
                steps.start(x, dy)
                run()
                got = [t.clone() for t in steps.results()]
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, w))
    finish()


@pytest.mark.parametrize("m,n,k", [(6144, 1500, 4096), (1024, 9000, 4096)])
def test_large_gradients_beside_one_another_are_exact(m, n, k):
    """Small whole numbers: sums below 2^24, whatever the order; and the next call's gradients, which take the same memory, are not early."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    whole = lambda *s: torch.randint(-3, 4, s, generator=gen, device="cuda").float()  # noqa: E731
    w = whole(m, k)
    weights = tuna_b200.fp8_quantize(w, "square")
    cases = [(whole(n, m), whole(n, k)) for _ in range(2)]
    dx, dw = torch.empty(n, k, device="cuda"), torch.empty(m, k, device="cuda")
    got = []
    for _ in range(3):
        for dy, x in cases:
            tuna_b200.fp8_matmul_backward(dy.half(), x.half(), None, *weights, dx, dw, m, n, k)
            got.append((dx.clone(), dw.clone()))
    finish()
    for i, (a, b) in enumerate(got):
        dy, x = cases[i % 2]
        assert torch.equal(a, dy @ w) and torch.equal(b, dy.T @ x)


def test_operands_of_two_types():
    """dy and x of different 16-bit types are quantized by launches of their own."""
    m, n, k = 272, 200, 400
    gen = torch.Generator(device="cuda").manual_seed(1)
    whole = lambda *s: torch.randint(-15, 16, s, generator=gen, device="cuda").float()  # noqa: E731
    dy, x, w = whole(n, m), whole(n, k), whole(m, k)
    for a, b in ((torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16)):
        dx, dw = torch.empty(n, k, device="cuda"), torch.empty(m, k, device="cuda")
        tuna_b200.fp8_matmul_backward(dy.to(a), x.to(b), None, *tuna_b200.fp8_quantize(w, "square"), dx, dw, m, n, k)
        finish()
        assert torch.equal(dx, dy @ w) and torch.equal(dw, dy.T @ x)


# ------------------------------------------------------------------ a kernel that lets its dependents start before it writes

def _late(names, args, call, outputs, graph):
    """What `names` say is written by the kernel right before the call."""
    call(args)
    finish()
    want = [o.clone() for o in outputs]
    assert all(torch.isfinite(w).all() and float(w.float().std()) > 1e-4 for w in want)
    late = {name: torch.zeros_like(args[name].view(torch.uint8)).view(args[name].dtype) for name in names}
    writer = torch.cuda._compile_kernel(LATE_WRITER, "late_writer")
    pairs = []
    for name in (names * 2)[:2]:
        src = args[name]
        pairs += [late[name].view(torch.uint8), src.view(torch.uint8), src.numel() * src.element_size()]

    def calls():
        writer(grid=(1, 1, 1), block=(256, 1, 1), args=pairs)
        call({**args, **late})

    run = calls
    if graph:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                calls()
        run = g.replay
    for _ in range(3):
        torch.cuda.synchronize()
        for t in late.values():
            t.view(torch.uint8).zero_()
        for o in outputs:
            o.fill_(float("nan"))
        torch.cuda.synchronize()
        run()
        finish()
        assert all(torch.equal(o, w) for o, w in zip(outputs, want))


M, F, K = 272, 144, 784


def _forward(n, gated, packed):
    gen = torch.Generator(device="cuda").manual_seed(n)
    q, s = tuna_b200.fp8_quantize(torch.randn(2 * F if gated else M, K, generator=gen, device="cuda"), "square")
    x = torch.randn(n, K, generator=gen, device="cuda", dtype=torch.bfloat16)
    args = {**(dict(zip(("x", "xs"), tuna_b200.fp8_quantize(x))) if packed else {"x": x}), "q": q, "s": s}
    out = torch.empty(n, F if gated else M, device="cuda")

    def call(a):
        if gated:
            tuna_b200.fp8_gated(a["x"], a.get("xs"), a["q"], a["s"], out, F, n, K)
        else:
            tuna_b200.fp8_matmul(a["x"], a.get("xs"), a["q"], a["s"], out, M, n, K)

    return args, call, [out]


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("packed", [True, False], ids=["codes", "numbers"])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("n", [1, 2, 16, 40, 64, 65, 300])
def test_tokens_of_the_kernel_before(n, gated, packed, graph):
    _late(["x", "xs"] if packed else ["x"], *_forward(n, gated, packed), graph)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("packed", [True, False], ids=["codes", "numbers"])
@pytest.mark.parametrize("gated", [False, True], ids=["plain", "gated"])
@pytest.mark.parametrize("n", [65, 300])
def test_weights_of_the_kernel_before(n, gated, packed, graph):
    """Above 64 tokens weights and their scales follow ordinary stream order, whatever the kernel before does about its dependents."""
    _late(["q", "s"], *_forward(n, gated, packed), graph)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("names", [["x", "dy"], ["q", "s"], ["xs", "z"]], ids=str)
@pytest.mark.parametrize("f,n,k", [(144, 20, 272), (144, 300, 272), (4096, 1200, 4096), (2048, 2500, 48)])
def test_operands_of_gradients_of_the_kernel_before(f, n, k, names, graph):
    gen = torch.Generator(device="cuda").manual_seed(n)
    q, s = tuna_b200.fp8_quantize(torch.randn(2 * f, k, generator=gen, device="cuda"), "square")
    x = torch.randn(n, k, generator=gen, device="cuda", dtype=torch.bfloat16)
    gated, packed = "z" in names, "xs" in names
    dy = torch.randn(n, f if gated else 2 * f, generator=gen, device="cuda", dtype=torch.bfloat16)
    args = {**(dict(zip(("x", "xs"), tuna_b200.fp8_quantize(x, "column"))) if packed else {"x": x}), "q": q, "s": s, "dy": dy}
    if gated:
        args["z"] = torch.randn(n, 2 * f, generator=gen, device="cuda", dtype=torch.bfloat16)
    dx, dw = torch.empty(n, k, device="cuda"), torch.empty(2 * f, k, device="cuda")

    def call(a):
        if gated:
            tuna_b200.fp8_gated_backward(a["dy"], a["z"], a["x"], a.get("xs"), a["q"], a["s"], dx, dw, f, n, k)
        else:
            tuna_b200.fp8_matmul_backward(a["dy"], a["x"], a.get("xs"), a["q"], a["s"], dx, dw, 2 * f, n, k)

    # the slow writer takes a few of them: what a large one would have it write for a second
    _late([name for name in names if args[name].numel() <= 1 << 20] or ["s"], args, call, [dx, dw], graph)


# ------------------------------------------------------------------ a process whose first call is captured

FIRST_CALL_CAPTURED = """
import torch, tuna_b200 as t
f, n, k = 272, 70, 400
x, dh = (torch.randn(n, c, device="cuda", dtype=torch.bfloat16) for c in (k, f))
w = torch.randn(2 * f, k, device="cuda")
h, z, dx, dw = (torch.empty(s, device="cuda", dtype=torch.bfloat16) for s in ((n, f), (n, 2 * f), (n, k), (2 * f, k)))
def step():
    q, s = t.fp8_quantize(w, "square")
    t.fp8_gated(x, None, q, s, h, f, n, k, z=z)
    t.fp8_gated_backward(dh, z, x, None, q, s, dx, dw, f, n, k)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    step()
g.replay()
torch.cuda.synchronize()
first = [v.clone() for v in (h, z, dx, dw)]
step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) and a.isfinite().all() for a, b in zip(first, (h, z, dx, dw)))
print("captured")
"""


def test_first_calls_of_a_process_can_be_captured():
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], capture_output=True, text=True, timeout=300, cwd=Path(__file__).resolve().parents[1], env=dict(os.environ))
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr
