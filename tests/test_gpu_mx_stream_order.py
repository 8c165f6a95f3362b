"""What a microscaled product sees of the kernels before it in its stream, without a synchronisation in between."""

import pytest
import torch

import tuna_b200
from tests.gpu_util import stream_ptr
from tuna_b200 import _lib

pytestmark = pytest.mark.gpu


def finish():
    torch.cuda.synchronize()
    assert _lib.load().tuna_check_device_status(stream_ptr()) == 0


# ------------------------------------------------------------------ one product's output is the next one's 16-bit input

# (m, n, k) of products that each read the first n * k numbers of the output before: tokens quantized in the launch (1 and 2 of
# them, 5 of few columns), in a launch before it (16, 40 and 300), folded tiles, low ones, pairs of CTAs
CHAINS = {
    "1": [(2048, 1, 2048)] * 6,
    "2": [(2048, 2, 2048)] * 6,
    "16": [(2048, 16, 2048)] * 6,
    "40": [(2048, 40, 2048)] * 6,
    "mixed": [(4096, 40, 1024), (4096, 16, 4096), (11000, 2, 4096), (4096, 1, 4096), (1024, 5, 512), (2048, 2, 2048), (4096, 1, 4096), (20000, 16, 256),
              (2048, 40, 4128), (512, 300, 256), (4096, 16, 4096), (4096, 1, 1056)],
}


class Chain:
    """Outputs go to two buffers in turn, so each is written again while the product that read it may still run."""

    def __init__(self, steps, dtype, grouped):
        gen = torch.Generator(device="cuda").manual_seed(len(steps))
        self.steps, self.grouped = steps, grouped
        self.weights = [tuna_b200.mx_quantize(torch.randn(m, k, generator=gen, device="cuda") * k ** -0.5) for m, _, k in steps]
        self.offsets = [torch.tensor([0, n], dtype=torch.int32, device="cuda") for _, n, _ in steps]
        _, n, k = steps[0]
        self.x = torch.empty(n, k, device="cuda", dtype=dtype)
        self.inputs = [torch.randn(n, k, generator=gen, device="cuda").to(dtype) for _ in range(3)]
        self.buffers = [torch.zeros(max(m * n for m, n, _ in steps), device="cuda", dtype=dtype) for _ in range(2)]
        self.kept = [torch.empty(m * n, device="cuda", dtype=dtype) for m, n, _ in steps]

    def run(self, between=None):
        x = self.x.view(-1)
        for i, (m, n, k) in enumerate(self.steps):
            assert x.numel() >= n * k
            o = self.buffers[i % 2][:m * n]
            q, s = self.weights[i]
            if self.grouped and i % 2:
                tuna_b200.mx_matmul_grouped(x[:n * k].view(n, k), None, q[None], s[None], self.offsets[i], o.view(n, m), m, n, k)
            else:
                tuna_b200.mx_matmul(x[:n * k].view(n, k), None, q, s, o.view(n, m), m, n, k)
            if between:
                between()
                self.kept[i].copy_(o)
                between()
            x = o
        return x


@pytest.mark.parametrize("grouped", [False, True], ids=["one", "experts"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("name", CHAINS)
def test_an_output_that_is_the_next_ones_tokens(name, dtype, grouped):
    """The same bits as with a synchronisation after every call, eager and replayed, with new inputs every time."""
    chain = Chain(CHAINS[name], dtype, grouped)
    want = []
    for x in chain.inputs:
        chain.x.copy_(x)
        want.append(chain.run(torch.cuda.synchronize).clone())
        assert all(torch.isfinite(o).all() and float(o.float().std()) > 1e-3 for o in chain.kept)
    assert not torch.equal(want[0], want[1])
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            chain.run()
    last = chain.buffers[(len(chain.steps) - 1) % 2][:want[0].numel()]
    for run in (chain.run, graph.replay):
        for _ in range(5):
            for x, w in zip(chain.inputs, want):
                for b in chain.buffers:
                    b.fill_(float("nan"))
                chain.x.copy_(x)
                run()
                got = last.clone()
                torch.cuda.synchronize()
                assert torch.equal(got, w)
    finish()


# ------------------------------------------------------------------ a kernel that lets its dependents start before it writes

# Lets its dependents start at once, writes only some 50 us later.
LATE_WRITER = """
extern "C" __global__ void late_writer(unsigned char *a, const unsigned char *a_src, int a_n, unsigned char *b, const unsigned char *b_src, int b_n)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const long long t0 = clock64();
    while (clock64() - t0 < 100000) { }
    for (int i = threadIdx.x; i < a_n; i += blockDim.x) a[i] = a_src[i];
    for (int i = threadIdx.x; i < b_n; i += blockDim.x) b[i] = b_src[i];
}
"""

M, K = 264, 800


def _operands(n, experts, packed):
    gen = torch.Generator(device="cuda").manual_seed(n)
    lead = (experts,) if experts else ()
    q, s = tuna_b200.mx_quantize(torch.randn(*lead, M, K, generator=gen, device="cuda"))
    x = torch.randn(n, K, generator=gen, device="cuda", dtype=torch.bfloat16)
    tokens = dict(zip(("x", "xs"), tuna_b200.mx_quantize(x))) if packed else {"x": x}
    args = {**tokens, "q": q, "s": s}
    if experts:
        args["offsets"] = torch.tensor([n * e // experts for e in range(experts + 1)], dtype=torch.int32, device="cuda")
    return args


def _call(args, o, n):
    if "offsets" in args:
        tuna_b200.mx_matmul_grouped(args["x"], args.get("xs"), args["q"], args["s"], args["offsets"], o, M, n, K)
    else:
        tuna_b200.mx_matmul(args["x"], args.get("xs"), args["q"], args["s"], o, M, n, K)


def _late(names, n, experts, packed, graph):
    """What `names` say is written by the kernel right before the call."""
    args = _operands(n, experts, packed)
    out, want = (torch.zeros(n, M, device="cuda") for _ in range(2))
    _call(args, want, n)
    finish()
    assert torch.isfinite(want).all() and float(want.std()) > 1
    late = {name: torch.zeros_like(args[name]) for name in names}
    writer = torch.cuda._compile_kernel(LATE_WRITER, "late_writer")
    pairs = []
    for name in (names * 2)[:2]:
        to, src = late[name], args[name]
        pairs += [to.view(torch.uint8), src.view(torch.uint8), src.numel() * src.element_size()]

    def calls():
        writer(grid=(1, 1, 1), block=(256, 1, 1), args=pairs)
        _call({**args, **late}, out, n)

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
            t.zero_()
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        run()
        finish()
        assert torch.equal(out, want)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("packed", [True, False], ids=["codes", "numbers"])
@pytest.mark.parametrize("n", [65, 100, 256, 300])
def test_weights_of_the_kernel_before(n, packed, graph):
    """Above 64 tokens weights and their scales follow ordinary stream order, whatever the kernel before does about its dependents."""
    _late(["q", "s"], n, 0, packed, graph)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("packed", [True, False], ids=["codes", "numbers"])
@pytest.mark.parametrize("n", [1, 16, 70, 300])
def test_experts_weights_of_the_kernel_before(n, packed, graph):
    _late(["q", "s"], n, 3, packed, graph)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("experts", [0, 3])
@pytest.mark.parametrize("packed", [True, False], ids=["codes", "numbers"])
@pytest.mark.parametrize("n", [1, 2, 16, 40, 64, 65, 300])
def test_tokens_of_the_kernel_before(n, packed, experts, graph):
    _late(["x", "xs"] if packed else ["x"], n, experts, packed, graph)


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
@pytest.mark.parametrize("packed", [True, False], ids=["codes", "numbers"])
@pytest.mark.parametrize("n", [1, 16, 40, 300])
def test_offsets_of_the_kernel_before(n, packed, graph):
    _late(["offsets"], n, 3, packed, graph)
