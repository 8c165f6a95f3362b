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
