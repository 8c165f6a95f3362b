"""Products of microscaled matrices on the GPU against sums in 64 bits, with the bound that mx_util derives."""

import numpy as np
import pytest
import torch

import tuna_b200
from tests.gpu_util import Guarded
from tests.mx_util import check_product, random_packed
from oracle import mx_oracle as mxo
from tuna_b200 import _lib

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def dev(*arrays):
    return [torch.from_numpy(a).cuda() for a in arrays]


def finish():
    torch.cuda.synchronize()
    assert _lib.load().tuna_check_device_status(torch.cuda.current_stream().cuda_stream) == 0


def product(m, n, k, seed=0, dtype=torch.float32, spread=3):
    (xq, xs), x = random_packed(n, k, 2 * seed + 1, spread)
    (wq, ws), w = random_packed(m, k, 2 * seed + 2, spread)
    hold = Guarded(n * m * dtype.itemsize, dtype, (n, m))
    tuna_b200.mx_matmul(*dev(xq, xs), *dev(wq, ws), hold.view, m, n, k)
    finish()
    assert hold.guards_intact()
    check_product(hold.view, x, w)
    return hold.view


@pytest.mark.parametrize("k", [32, 64, 96, 128, 160, 256, 288, 512, 4096])
def test_one_token(k):
    product(128, 1, k, seed=k)


@pytest.mark.parametrize("m", [8, 16, 120, 128, 136, 1000, 4096])
def test_output_features(m):
    product(m, 3, 544, seed=m)


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 300, 513])
def test_tokens(n):
    product(264, n, 800, seed=n, dtype=torch.bfloat16)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,k", [(4096, 1, 4096), (1000, 43, 4128), (6144, 256, 1024), (520, 130, 14336), (20000, 16, 512), (2048, 700, 2048), (40, 2000, 96)])
def test_sizes_and_types(m, n, k, dtype):
    product(m, n, k, seed=m + n, dtype=dtype)


def test_single_products_are_exact():
    """One column of x is not zero: the outputs are w's numbers, so no row, column or scale is taken for another."""
    m, n, k = 384, 40, 1056
    rng = np.random.default_rng(5)
    (wq, ws), w = random_packed(m, k, 6, spread=8)
    codes = np.zeros((n, k), dtype=np.uint8)
    at = rng.permutation(k)[:n]
    codes[np.arange(n), at] = 2  # 1.0
    scales = rng.integers(120, 135, (n, k // 32), dtype=np.uint8)
    o = torch.full((n, m), float("nan"), device="cuda")
    tuna_b200.mx_matmul(*dev(*mxo.pack(codes, scales)), *dev(wq, ws), o, m, n, k)
    finish()
    want = w[:, at].T * 2.0 ** (scales[np.arange(n), at // 32].astype(float) - 127)[:, None]
    assert np.array_equal(o.double().cpu().numpy(), want)


def test_scales_of_every_size_and_nan():
    """Scales from 2^-60 to 2^60 on either side; a NaN scale spoils its own row's or token's outputs and no others."""
    m, n, k = 256, 20, 512
    (xq, xs), x = random_packed(n, k, 1, spread=60)
    (wq, ws), w = random_packed(m, k, 2, spread=0)
    xs[2, 7, 1] = 255
    x[7, 9 * 32:10 * 32] = np.nan
    o = torch.empty(n, m, device="cuda")
    tuna_b200.mx_matmul(*dev(xq, xs), *dev(wq, ws), o, m, n, k)
    finish()
    check_product(o, x, w)
    ws[3, 100, 3] = 255
    w[100, 15 * 32:] = np.nan
    tuna_b200.mx_matmul(*dev(xq, xs), *dev(wq, ws), o, m, n, k)
    finish()
    check_product(o, x, w)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("m,n,k", [(128, 1, 32), (512, 5, 2080), (1024, 40, 4096), (256, 300, 768)])
def test_tokens_in_16_bits_are_quantized_by_the_call(m, n, k, dtype):
    x = torch.randn(n, k, device="cuda").to(dtype)
    x[:, 3] *= 30
    (wq, ws), w = random_packed(m, k, 4)
    o = torch.empty(n, m, device="cuda", dtype=dtype)
    q, s = dev(wq, ws)
    tuna_b200.mx_matmul(x, None, q, s, o, m, n, k)
    finish()
    codes, scales = mxo.quantize(x.double().cpu().numpy())
    check_product(o, mxo.decode(codes, scales), w)
    o2 = torch.empty_like(o)
    tuna_b200.mx_matmul(*tuna_b200.mx_quantize(x), q, s, o2, m, n, k)
    assert torch.equal(o, o2)


@pytest.mark.parametrize("n", [3, 24])
def test_runs_agree_bit_for_bit_in_any_workspace(n):
    m, k = 2000, 8192
    (wq, ws), _ = random_packed(m, k, 2)
    q, s = dev(wq, ws)
    x = torch.randn(n, k, device="cuda", dtype=torch.float16)
    outs = []
    for fill in (None, 0, 255):
        work = None if fill is None else torch.full((1 << 20,), fill, dtype=torch.uint8, device="cuda")
        o = torch.full((n, m), float("nan"), device="cuda")
        tuna_b200.mx_matmul(x, None, q, s, o, m, n, k, workspace=work)
        outs.append(o)
    finish()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("n", [1, 2, 5, 7, 16, 40])
def test_tokens_with_infinities_and_nan_spoil_only_their_own_outputs(n):
    m, k = 200, 1184
    (wq, ws), w = random_packed(m, k, 8)
    x = torch.randn(n, k, device="cuda", dtype=torch.bfloat16)
    x[0, 5] = float("inf")
    if n > 1:
        x[n - 1, k - 1] = float("nan")
    o = torch.empty(n, m, device="cuda")
    tuna_b200.mx_matmul(x, None, *dev(wq, ws), o, m, n, k)
    finish()
    assert torch.isnan(o[0]).all() and torch.isnan(o[n - 1]).all()
    check_product(o, mxo.decode(*mxo.quantize(x.double().cpu().numpy())), w)


@pytest.mark.parametrize("m", [8, 24, 264, 1184, 2368, 4736, 9472, 18944, 19000])
def test_row_tiles_of_every_height(m):
    """Up to 16 tokens: one to 128 rows a tile, folded four ways, two ways and not, with and without a remainder."""
    for n, k in ((1, 416), (9, 1312)):
        product(m, n, k, seed=m)
    x = torch.randn(3, 672, device="cuda", dtype=torch.float16)
    (wq, ws), w = random_packed(m, 672, 5)
    o = torch.empty(3, m, device="cuda")
    tuna_b200.mx_matmul(x, None, *dev(wq, ws), o, m, 3, 672)
    finish()
    check_product(o, mxo.decode(*mxo.quantize(x.double().cpu().numpy())), w)


@pytest.mark.parametrize("n", [17, 33, 49, 65, 97, 129, 145, 161, 177, 193, 225, 257, 353, 400, 530])
def test_token_tiles_of_every_width(n):
    product(2600, n, 320, seed=n)


def test_an_output_of_more_than_2_31_elements():
    m, n, k = 65536, 33000, 32
    (xq, xs), x = random_packed(n, k, 1)
    (wq, ws), w = random_packed(m, k, 2)
    o = torch.empty(n, m, device="cuda", dtype=torch.bfloat16)
    tuna_b200.mx_matmul(*dev(xq, xs, wq, ws), o, m, n, k)
    finish()
    for rows in (slice(0, 3), slice(16000, 16003), slice(n - 300, n)):
        check_product(o[rows], x[rows], w)


# ------------------------------------------------------------------ experts

def grouped(counts, m, k, *, before=0, behind=0, dtype=torch.float32, seed=0, quantized=True, offsets=None):
    e, n = len(counts), before + sum(counts) + behind
    ends = before + np.cumsum([0] + list(counts))
    mats = [random_packed(m, k, 100 * seed + i) for i in range(e)]
    q, s = dev(np.stack([p[0][0] for p in mats]), np.stack([p[0][1] for p in mats]))
    hold = Guarded(n * m * dtype.itemsize, dtype, (n, m))
    hold.view.fill_(7.0)
    off = torch.from_numpy(ends.astype(np.int32)).cuda()
    if quantized:
        (xq, xs), x = random_packed(n, k, 100 * seed + 99)
        tuna_b200.mx_matmul_grouped(*dev(xq, xs), q, s, off, hold.view, m, n, k)
    else:
        t = torch.randn(n, k, device="cuda", dtype=torch.bfloat16)
        x = mxo.decode(*mxo.quantize(t.double().cpu().numpy()))
        tuna_b200.mx_matmul_grouped(t, None, q, s, off, hold.view, m, n, k)
    finish()
    assert hold.guards_intact()
    for i in range(e):
        if counts[i]:
            check_product(hold.view[ends[i]:ends[i + 1]], x[ends[i]:ends[i + 1]], mats[i][1])
    assert (hold.view[:before] == 7).all() and (hold.view[ends[-1]:] == 7).all(), "rows of no expert are left as they were"


@pytest.mark.parametrize("counts", [[1], [0, 1], [5, 0, 3], [0, 0, 0, 9], [1] * 40, [17, 16, 15, 1, 0, 33], [200, 3, 0, 129, 64], [0, 0], [700, 1]], ids=str)
def test_experts(counts):
    grouped(counts, 264, 544, seed=len(counts))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("quantized", [True, False])
def test_experts_in_a_larger_buffer(dtype, quantized):
    grouped([3, 0, 21, 7], 136, 416, before=5, behind=9, dtype=dtype, quantized=quantized)


def test_decreasing_offsets_of_many_experts():
    """Every offset counts as the largest up to it: 70 experts, of which most get nothing."""
    m, n, k, experts = 64, 90, 96, 70
    rng = np.random.default_rng(7)
    offsets = rng.integers(-20, n + 20, experts + 1).astype(np.int32)
    offsets[:40] = rng.integers(-5, 30, 40)
    mats = [random_packed(m, k, i) for i in range(experts)]
    q, s = dev(np.stack([p[0][0] for p in mats]), np.stack([p[0][1] for p in mats]))
    (xq, xs), x = random_packed(n, k, 999)
    o = torch.full((n, m), 7.0, device="cuda")
    tuna_b200.mx_matmul_grouped(*dev(xq, xs), q, s, torch.from_numpy(offsets).cuda(), o, m, n, k)
    finish()
    ends = np.maximum.accumulate(np.clip(offsets, 0, n))
    for e in range(experts):
        if ends[e] < ends[e + 1]:
            check_product(o[ends[e]:ends[e + 1]], x[ends[e]:ends[e + 1]], mats[e][1])
    assert (o[:ends[0]] == 7).all() and (o[ends[-1]:] == 7).all()


def test_many_experts():
    rng = np.random.default_rng(0)
    grouped(list(rng.integers(0, 4, 1024)), 16, 96, seed=3)


def test_odd_numbers_of_tokens_shift_every_experts_rows():
    grouped([1, 2, 3, 5, 7, 11, 13], 1000, 1056, before=1, seed=4)


def test_experts_without_tokens_at_all():
    (wq, ws), _ = random_packed(128, 256, 1)
    q, s = dev(wq[None], ws[None])
    tuna_b200.mx_matmul_grouped(torch.empty(0, 256, device="cuda", dtype=torch.bfloat16), None, q, s, torch.zeros(2, dtype=torch.int32, device="cuda"),
                                torch.empty(0, 128, device="cuda"), 128, 0, 256)
    finish()


@pytest.mark.parametrize("offsets", [[0, 99, 20], [-5, 3, 8], [4, 2, 6], [7, 3, 1], [-2147483648, 0, 2147483647]], ids=str)
def test_offsets_outside_the_tokens_stay_inside_the_output(offsets):
    m, n, k = 128, 8, 256
    mats = [random_packed(m, k, i) for i in range(2)]
    q, s = dev(np.stack([p[0][0] for p in mats]), np.stack([p[0][1] for p in mats]))
    (xq, xs), x = random_packed(n, k, 9)
    hold = Guarded(n * m * 4, torch.float32, (n, m))
    hold.view.fill_(7.0)
    tuna_b200.mx_matmul_grouped(*dev(xq, xs), q, s, torch.tensor(offsets, dtype=torch.int32, device="cuda"), hold.view, m, n, k)
    finish()
    assert hold.guards_intact()
    clamped = np.maximum.accumulate(np.clip(offsets, 0, n))
    covered = np.zeros(n, dtype=bool)
    for e in range(2):
        covered[clamped[e]:max(clamped[e], clamped[e + 1])] = True
    assert (hold.view[torch.from_numpy(~covered).cuda()] == 7).all()
    for r in np.flatnonzero(covered):
        e = next(e for e in range(2) if clamped[e] <= r < clamped[e + 1])
        check_product(hold.view[r:r + 1], x[r:r + 1], mats[e][1])


@pytest.mark.parametrize("n", [1, 2, 16, 17, 19, 43, 130, 515])
@pytest.mark.parametrize("first,last", [(1, 4), (2, 3), (3, 5), (0, 2)])
def test_column_ranges_are_views(n, first, last):
    """Columns 256 first .. 256 last of both operands, which start on 4 bytes where the tokens' scales do."""
    m, k = 264, 1216
    (wq, ws), w = random_packed(m, k, 5)
    (xq, xs), x = random_packed(n, k, 6)
    a, b = 256 * first, min(k, 256 * last)
    wq, ws, xq, xs = dev(wq, ws, xq, xs)
    words = slice(2 * first, 2 * first + -(-(b - a) // 128))
    o = torch.empty(n, m, device="cuda")
    tuna_b200.mx_matmul(xq[first:last], xs[words], wq[first:last], ws[words], o, m, n, b - a)
    finish()
    check_product(o, x[:, a:b], w[:, a:b])
    if first:
        off = torch.tensor([0, n // 2, n], dtype=torch.int32, device="cuda")
        two = torch.empty_like(o)
        tuna_b200.mx_matmul_grouped(xq[first:last], xs[words], wq[first:last].expand(2, -1, -1, -1).contiguous(), ws[words].expand(2, -1, -1, -1).contiguous(), off, two,
                                    m, n, b - a)
        finish()
        check_product(two, x[:, a:b], w[:, a:b])


# ------------------------------------------------------------------ streams, graphs, devices, a layer

def test_a_mixture_layer_from_activations_to_outputs():
    """Tokens sorted by expert -> gate+up -> gated activation -> down: every call as a program makes it, one after another."""
    experts, hidden, inter, tokens = 6, 512, 768, 50
    rng = np.random.default_rng(1)
    choice = np.sort(rng.integers(0, experts, tokens))
    off = torch.from_numpy(np.searchsorted(choice, np.arange(experts + 1)).astype(np.int32)).cuda()
    up = tuna_b200.mx_quantize(torch.randn(experts, 2 * inter, hidden, device="cuda") * hidden ** -0.5)
    down = tuna_b200.mx_quantize(torch.randn(experts, hidden, inter, device="cuda") * inter ** -0.5)
    x = torch.randn(tokens, hidden, device="cuda", dtype=torch.bfloat16)
    h = torch.empty(tokens, 2 * inter, device="cuda", dtype=torch.bfloat16)
    o = torch.empty(tokens, hidden, device="cuda", dtype=torch.bfloat16)
    tuna_b200.mx_matmul_grouped(x, None, *up, off, h, 2 * inter, tokens, hidden)
    a = torch.nn.functional.silu(h[:, :inter].float()) * h[:, inter:].float()
    a = a.to(torch.bfloat16)
    tuna_b200.mx_matmul_grouped(a, None, *down, off, o, hidden, tokens, inter)
    finish()

    def numbers(t):
        return mxo.decode(*mxo.quantize(t.double().cpu().numpy()))

    def matrix(pair, e, rows, k):
        w = torch.empty(rows, k, device="cuda")
        tuna_b200.mx_dequant(pair[0][e], pair[1][e], w, rows, k)
        return w.double().cpu().numpy()

    for e in range(experts):
        rows = np.flatnonzero(choice == e)
        if len(rows):
            check_product(h[rows], numbers(x[rows]), matrix(up, e, 2 * inter, hidden))
            check_product(o[rows], numbers(a[rows]), matrix(down, e, hidden, inter))


def test_two_graphs_of_one_stream_replayed_side_by_side():
    m, n, k = 1024, 16, 8192
    cases = []
    for i in range(2):
        (xq, xs), x = random_packed(n, k, 10 + i)
        (wq, ws), w = random_packed(m, k, 20 + i)
        cases.append((dev(xq, xs, wq, ws), torch.zeros(n, m, device="cuda"), x, w))
    graphs = []
    side = torch.cuda.Stream()
    for args, o, _, _ in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            for _ in range(3):
                tuna_b200.mx_matmul(*args, o, m, n, k)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(30):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    finish()
    for _, o, x, w in cases:
        check_product(o, x, w)


@pytest.mark.parametrize("n", [2, 24])
def test_graphs_with_tokens_in_16_bits(n):
    """Captured calls that quantize their tokens, replayed with new ones side by side with eager calls on another stream."""
    m, k = 1024, 4096
    (wq, ws), w = random_packed(m, k, 2)
    q, s = dev(wq, ws)
    xs = [torch.zeros(n, k, device="cuda", dtype=torch.float16) for _ in range(2)]
    outs = [torch.zeros(n, m, device="cuda") for _ in range(3)]
    graphs = []
    for x, o in zip(xs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            tuna_b200.mx_matmul(x, None, q, s, o, m, n, k)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    eager = torch.randn(n, k, device="cuda", dtype=torch.float16)
    for round_ in range(5):
        for x in xs:
            x.normal_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            tuna_b200.mx_matmul(eager, None, q, s, outs[2], m, n, k)
        finish()
        for x, o in zip(xs + [eager], outs):
            check_product(o, mxo.decode(*mxo.quantize(x.double().cpu().numpy())), w)


@pytest.mark.parametrize("experts,captured", [(3, False), (3, True), (70, True)])
def test_offsets_written_right_before_the_call(experts, captured):
    """A kernel writes the offsets, the call quantizes its tokens, and the next kernel writes other offsets, without a wait in between."""
    m, n, k, rounds = 512, 80, 1024, 6
    rng = np.random.default_rng(experts)
    q, s = tuna_b200.mx_quantize(torch.randn(experts, m, k, device="cuda"))
    x = torch.randn(n, k, device="cuda", dtype=torch.bfloat16)
    xq, xs = tuna_b200.mx_quantize(x)
    counts = [torch.from_numpy(np.diff(np.sort(rng.integers(0, n + 1, experts - 1)), prepend=0, append=n).astype(np.int32)).cuda() for _ in range(rounds)]
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    off = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    outs = [torch.full((n, m), 7.0, device="cuda") for _ in range(rounds)]

    def run():
        for c, o in zip(counts, outs):
            torch.cumsum(torch.cat([zero, c]), 0, dtype=torch.int32, out=off)
            tuna_b200.mx_matmul_grouped(x, None, q, s, off, o, m, n, k)

    if captured:
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        for _ in range(5):
            for o in outs:
                o.fill_(7.0)
            graph.replay()
    else:
        for _ in range(5):
            run()
    finish()
    for c, o in zip(counts, outs):
        torch.cumsum(torch.cat([zero, c]), 0, dtype=torch.int32, out=off)
        want = torch.empty_like(o)
        torch.cuda.synchronize()
        tuna_b200.mx_matmul_grouped(xq, xs, q, s, off, want, m, n, k)
        finish()
        assert torch.equal(o, want)


def test_calls_on_two_streams_at_once():
    m, n, k = 1024, 16, 4096
    (xq, xs), x = random_packed(n, k, 1)
    (wq, ws), w = random_packed(m, k, 2)
    args = dev(xq, xs, wq, ws)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [torch.zeros(n, m, device="cuda") for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, o in zip(streams, outs):
            with torch.cuda.stream(st):
                tuna_b200.mx_matmul(*args, o, m, n, k)
    finish()
    for o in outs:
        check_product(o, x, w)


def test_dependent_calls_without_a_wait_in_between():
    """Weights and tokens quantized right before the product, overwritten right after it, over and over on one stream."""
    m, n, k = 768, 33, 2048
    gen = torch.Generator(device="cuda").manual_seed(1)
    pairs = [(torch.randn(m, k, generator=gen, device="cuda"), torch.randn(n, k, generator=gen, device="cuda", dtype=torch.float16)) for _ in range(4)]
    want = []
    for w, x in pairs:
        o = torch.empty(n, m, device="cuda")
        torch.cuda.synchronize()
        q, s = tuna_b200.mx_quantize(w)
        torch.cuda.synchronize()
        tuna_b200.mx_matmul(x, None, q, s, o, m, n, k)
        torch.cuda.synchronize()
        want.append(o)
    wbuf, xbuf = torch.empty(m, k, device="cuda"), torch.empty(n, k, device="cuda", dtype=torch.float16)
    got = [torch.empty(n, m, device="cuda") for _ in range(20)]
    for i, o in enumerate(got):
        wbuf.copy_(pairs[i % 4][0])
        xbuf.copy_(pairs[i % 4][1])
        q, s = tuna_b200.mx_quantize(wbuf)
        if i % 2:
            tuna_b200.mx_matmul(xbuf, None, q, s, o, m, n, k)
        else:
            tuna_b200.mx_matmul(*tuna_b200.mx_quantize(xbuf), q, s, o, m, n, k)
        q.zero_()
    finish()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 4])


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_a_device_that_is_not_the_current_one():
    m, n, k = 256, 5, 512
    (xq, xs), x = random_packed(n, k, 1)
    (wq, ws), w = random_packed(m, k, 2)
    o = torch.empty(n, m, device="cuda:1")
    tuna_b200.mx_matmul(*(t.to("cuda:1") for t in dev(xq, xs, wq, ws)), o, m, n, k)
    torch.cuda.synchronize(1)
    check_product(o, x, w)


def test_calls_checked_in_python_are_the_same_calls(monkeypatch):
    """Without the native front every call goes through the checks and the binding of mx.py."""
    m, n, k = 264, 21, 544
    w = torch.randn(3, m, k, device="cuda")
    x = torch.randn(n, k, device="cuda", dtype=torch.float16)
    off = torch.tensor([0, 4, 4, 19], dtype=torch.int32, device="cuda")

    def calls():
        q, s = tuna_b200.mx_quantize(w)
        xq, xs = tuna_b200.mx_quantize(x)
        outs = [q, s, xq, xs] + [torch.zeros(n, m, device="cuda") for _ in range(4)] + [torch.empty(m, k, device="cuda", dtype=torch.bfloat16)]
        tuna_b200.mx_matmul(x, None, q[0], s[0], outs[4], m, n, k)
        tuna_b200.mx_matmul(xq, xs, q[0], s[0], outs[5], m, n, k)
        tuna_b200.mx_matmul_grouped(x, None, q, s, off, outs[6], m, n, k)
        tuna_b200.mx_matmul_grouped(xq, xs, q, s, off, outs[7], m, n, k)
        tuna_b200.mx_dequant(q[1], s[1], outs[8], m, k)
        finish()
        return outs

    native = calls()
    monkeypatch.setattr(tuna_b200.mx, "_front", lambda: tuna_b200.mx._NoFront)
    for a, b in zip(native, calls()):
        assert torch.equal(a, b)


def test_errors_of_a_launch_are_raised_by_the_native_front():
    x = torch.randn(5 * 256 + 8, device="cuda", dtype=torch.float16)[4:4 + 4 * 256].view(4, 256)  # 8 bytes off
    (wq, ws), _ = random_packed(128, 256, 1)
    with pytest.raises(tuna_b200.TunaError) as e:
        tuna_b200.mx_matmul(x, None, *dev(wq, ws), torch.empty(4, 128, device="cuda"), 128, 4, 256)
    assert e.value.status == -3
    with pytest.raises(tuna_b200.TunaError):
        tuna_b200.mx_quantize(x)


def test_refusals():
    m, n, k = 128, 4, 256
    (xq, xs), _ = random_packed(n, k, 1)
    (wq, ws), _ = random_packed(m, k, 2)
    xq, xs, wq, ws = dev(xq, xs, wq, ws)
    o = torch.empty(n, m, device="cuda")
    off = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in ((xq, xs, wq, ws, o, m, n, 480), (xq, xs, wq, ws, o, m, n + 1, k), (xq, xs, wq, ws[:1], o, m, n, k), (xq, xs, wq, ws, o.t(), m, n, k),
                (xq, xs, wq, ws, o.cpu(), m, n, k), (xq, xs[:, :, ::2], wq, ws, o, m, n, k)):
        with pytest.raises(ValueError):
            tuna_b200.mx_matmul(*bad)
    with pytest.raises(TypeError):
        tuna_b200.mx_matmul(xq, xs, wq, ws, o.double(), m, n, k)
    with pytest.raises(TypeError):
        tuna_b200.mx_matmul(torch.empty(n, k, device="cuda"), None, wq, ws, o, m, n, k)
    with pytest.raises(tuna_b200.TunaError):
        tuna_b200.mx_matmul(torch.empty(40, k, device="cuda", dtype=torch.bfloat16), None, wq, ws, torch.empty(40, m, device="cuda"), m, 40, k,
                            workspace=torch.zeros(64, dtype=torch.uint8, device="cuda"))
    x16, o16, need = torch.zeros(40, k, device="cuda", dtype=torch.bfloat16), torch.empty(40, m, device="cuda"), 40 * 264
    for bad in (torch.zeros(need, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8, device="cuda").expand(need),
                torch.zeros(2 * need, dtype=torch.uint8, device="cuda")[::2]):  # off the GPU, not as long as it says, with gaps
        with pytest.raises(ValueError, match="workspace"):
            tuna_b200.mx_matmul(x16, None, wq, ws, o16, m, 40, k, workspace=bad)
        with pytest.raises(ValueError, match="workspace"):
            tuna_b200.mx_matmul_grouped(x16, None, wq[None], ws[None], off, o16, m, 40, k, workspace=bad)
    with pytest.raises(TypeError, match="workspace"):
        tuna_b200.mx_matmul(x16, None, wq, ws, o16, m, 40, k, workspace=4096)
    with pytest.raises(ValueError):
        tuna_b200.mx_matmul_grouped(xq, xs, wq, ws, off, o, m, n, k)  # no leading dimension
    with pytest.raises(TypeError):
        tuna_b200.mx_matmul_grouped(xq, xs, wq[None], ws[None], off.long(), o, m, n, k)
    with pytest.raises(ValueError):
        tuna_b200.mx_matmul_grouped(xq, xs, wq[None], ws[None], off[:1], o, m, n, k)
    with pytest.raises(ValueError):
        tuna_b200.mx_matmul_grouped(xq, xs, wq[None], ws[None], off.cpu(), o, m, n, k)
