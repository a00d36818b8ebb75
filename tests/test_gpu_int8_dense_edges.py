"""The 8-bit integer products where they can go wrong: waits that run out, and every kernel over several tiles."""
from __future__ import annotations

import threading

import pytest
import torch

import conftest  # noqa: F401
from qcc_b200 import _lib
from qcc_b200.runtime.block_norm import BlockNorm, residual_norm
from qcc_b200.runtime.int8_dense import Int8GatedFFN, int8_gated_linear, int8_linear, quantize_rows
from test_gpu_int8_dense import check_gated, check_linear, operands, product64

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture
def no_waiting():
    """Launches made inside give up at once unless their copies are there already."""
    lib = _lib.library()
    assert lib.qcc_set_wait_limit(0) == _lib.OK
    yield
    lib.qcc_set_wait_limit(2_000_000_000)
    torch.cuda.synchronize()


# The stream kernel alone, with its columns split over a cluster, with 32, 64 and 128 tokens a tile; and CTA pairs with
# one and with several tiles (more than 74), short and long columns.
@pytest.mark.parametrize("tokens,rows,cols", [(1, 40000, 700), (3, 256, 9000), (30, 1000, 4000), (60, 500, 100),
                                              (100, 5120, 17408), (600, 4000, 2000), (1100, 6000, 1500),
                                              (1100, 6000, 300)])
@pytest.mark.parametrize("gated", [False, True])
def test_a_wait_that_runs_out_leaves_nan(tokens, rows, cols, gated, request):
    call = int8_gated_linear if gated else int8_linear
    xq, xs, wq, ws = operands(tokens, rows, cols)
    channels = rows // 2 if gated else rows
    want = call(xq, xs, wq, ws, out_dtype=FP32)
    request.getfixturevalue("no_waiting")
    flat = torch.full((tokens * channels + 64,), 7.0, device="cuda")
    got = call(xq, xs, wq, ws, out=flat[:tokens * channels].view(tokens, channels))
    torch.cuda.synchronize()
    assert bool((flat[tokens * channels:] == 7).all())
    lost = got.isnan()
    assert bool(lost.any()) and torch.equal(got[~lost], want[~lost])
    # With the ordinary bound again nothing of the launch that gave up arrives later.
    _lib.library().qcc_set_wait_limit(2_000_000_000)
    for _ in range(3):
        assert torch.equal(call(xq, xs, wq, ws, out_dtype=FP32), want)


def test_layer_of_more_than_32768_neurons():
    hidden, inner, tokens = 64, 36864, 5
    gen = torch.Generator().manual_seed(0)

    def make(*shape, scale):
        return (torch.randn(shape, generator=gen) * scale).to(BF16).cuda()

    gate, up, down = make(inner, hidden, scale=0.1), make(inner, hidden, scale=0.1), make(hidden, inner, scale=0.01)
    x = make(tokens, hidden, scale=1.0)
    for ffn in (Int8GatedFFN.from_weights(gate, up, down),
                Int8GatedFFN.from_weights(gate, up, down.t().contiguous(), transposed_down=True)):
        stored = ffn.gate_up(x, out_dtype=BF16)
        hq, hs = quantize_rows(stored)
        check_linear(ffn(x), product64(hq, hs, ffn.down.weight, ffn.down.scale))
        dense = (torch.nn.functional.silu(x.double() @ gate.double().t()) * (x.double() @ up.double().t())) \
            @ down.double().t()
        # Each of the four roundings to int8 is half a step, 1/254 of a row's largest value, at most.
        assert float((ffn(x).double() - dense).norm() / dense.norm()) < 0.05


@pytest.mark.parametrize("tokens,cols", [(3, 40), (40, 1500), (130, 200)])
def test_scales_at_the_ends_of_fp32(tokens, cols):
    """The product of the scales leaves the normal range, the result does not."""
    rows = 96
    xq, _, wq, _ = operands(tokens, rows, cols)
    xq[0, 0], wq[0] = 0, 0  # sums of 0 under scales whose product is infinite
    exponents = torch.tensor([-126.0, -120.0, -100.0, -75.0, -40.0, 0.0, 40.0, 70.0, 100.0], device="cuda")
    xs = 1.3 * 2.0 ** exponents[torch.arange(tokens, device="cuda") % 9]
    ws = 1.7 * 2.0 ** exponents[(torch.arange(rows, device="cuda") * 5 + 2) % 9]
    xs[1] = 0.0
    sums = (xq.double() @ wq.double().t())
    want = sums * xs.double()[:, None] * ws.double()
    y = int8_linear(xq, xs, wq, ws, out_dtype=FP32)
    largest, least = torch.finfo(FP32).max, 2.0 ** -126
    over = want.abs() > largest
    assert bool((y[over].double() == torch.sign(want[over]) * float("inf")).all())
    # Three roundings (the sum's, and one a scale), and half a step of the smallest numbers.
    bound = 3 * 2.0 ** -24 * want.abs() * (1 + 2.0 ** -20) + 2.0 ** -149
    assert bool(((y.double() - want).abs() <= bound)[~over].all())
    assert bool((y[:, 0] == 0).all()) and bool((y[1] == 0).all())
    assert int(((want.abs() >= least) & (xs.double()[:, None] * ws.double() < least)).sum()) > 0
    # Gate and up rows alike: the gate ordinary, the up rows at the ends.
    gate_ws = torch.full((rows // 2,), 2.0 ** -14, device="cuda")
    ws2 = torch.cat([gate_ws, ws[rows // 2:]])
    xs2 = torch.where(exponents[torch.arange(tokens, device="cuda") % 9] <= -100.0, xs, torch.ones_like(xs))
    both = sums * xs2.double()[:, None] * ws2.double()
    g, u = both[:, :rows // 2], both[:, rows // 2:]
    h = int8_gated_linear(xq, xs2, wq, ws2, out_dtype=FP32)
    fits = (g * torch.sigmoid(g) * u).abs() <= largest
    fits &= u.abs() <= largest
    check_gated(h[fits], g[fits], u[fits])


@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_silu_far_below_zero(tokens):
    """silu keeps its value down to fp32's smallest numbers, and large up projections show it."""
    channels = 9000  # of pair tiles at 300 tokens
    xq = torch.zeros((tokens, 16), dtype=torch.int8, device="cuda")
    xq[:, 0], xq[:, 1] = -127, 127
    wq = torch.zeros((2 * channels, 16), dtype=torch.int8, device="cuda")
    wq[:channels, 0], wq[channels:, 1] = 127, 127
    depth = torch.linspace(70.0, 101.0, channels, device="cuda")
    ws = torch.cat([depth / 127 ** 2, torch.full((channels,), 1e30 / 127 ** 2, device="cuda")])
    xs = torch.ones(tokens, device="cuda")
    both = product64(xq, xs, wq, ws)
    g, u = both[:, :channels], both[:, channels:]
    h = int8_gated_linear(xq, xs, wq, ws, out_dtype=FP32)
    want = g * torch.sigmoid(g) * u
    # As in the products' tests, with exp's smallest numbers off by 2^-149 at most instead of an error of 2^-119 |u|.
    bound = want.abs() * (2.0 ** -24 + (16 + 4 * g.abs()) * 2.0 ** -24 * 1.01) + 2.0 ** -148 * g.abs() * u.abs()
    assert bool(((h.double() - want).abs() <= bound).all())
    assert bool((h != 0).all())


# By the kernels' rules on 148 SMs: CTA pairs with one tile and with several (more than 74, so that both accumulators,
# the stages across tiles and groups of eight token tiles come round), with tiles of few tokens at the end (1800: eight
# of 225) and fewer column blocks than stages; and the stream kernel with tiles of 128 tokens, one and two of them.
LINEAR = [(300, 5000, 700), (1111, 5000, 900), (2600, 2100, 300), (1800, 2600, 200), (4096, 1300, 130),
          (65, 5120, 17408), (128, 5120, 17408), (250, 5120, 17408)]
GATED = [(300, 2500, 700), (1111, 2500, 900), (2600, 1100, 300), (1800, 1300, 200), (4096, 700, 130),
         (65, 5200, 5120), (128, 5200, 5120)]


@pytest.mark.parametrize("tokens,rows,cols", LINEAR)
def test_linear_over_several_tiles(tokens, rows, cols):
    xq, xs, wq, ws = operands(tokens, rows, cols)
    want = product64(xq, xs, wq, ws)
    bias = torch.randn(rows, generator=torch.Generator().manual_seed(3)).cuda()
    for dtype in (BF16, FP16, FP32):
        flat = torch.full((tokens * rows + 64,), 7.0, dtype=dtype, device="cuda")
        y = int8_linear(xq, xs, wq, ws, bias=bias, out=flat[:tokens * rows].view(tokens, rows))
        check_linear(y, want, bias)
        assert bool((flat[tokens * rows:] == 7).all())
        assert torch.equal(int8_linear(xq, xs, wq, ws, bias=bias, out_dtype=dtype), y)
    # A token's result does not depend on the batch or the kernel that it comes in.
    for t in (1, 40, 65):
        part = int8_linear(xq[-t:], xs[-t:], wq, ws, bias=bias, out_dtype=FP32)
        assert torch.equal(part, y[-t:])


@pytest.mark.parametrize("tokens,rows,cols", GATED)
def test_gated_over_several_tiles(tokens, rows, cols):
    xq, xs, wq, ws = operands(tokens, 2 * rows, cols)
    both = product64(xq, xs, wq, ws)
    for dtype in (BF16, FP16, FP32):
        flat = torch.full((tokens * rows + 64,), 7.0, dtype=dtype, device="cuda")
        h = int8_gated_linear(xq, xs, wq, ws, out=flat[:tokens * rows].view(tokens, rows))
        check_gated(h, both[:, :rows], both[:, rows:])
        assert bool((flat[tokens * rows:] == 7).all())
        assert torch.equal(int8_gated_linear(xq, xs, wq, ws, out_dtype=dtype), h)
    for t in (1, 40, 65):
        assert torch.equal(int8_gated_linear(xq[-t:], xs[-t:], wq, ws, out_dtype=FP32), h[-t:])


def test_outputs_beyond_2_to_the_31_elements():
    """The most tokens that are taken, with outputs whose offsets pass 32 bits."""
    tokens, rows, cols = 1 << 20, 2100, 20
    xq, xs, wq, ws = operands(70, rows, cols)
    xq = torch.cat([xq.new_zeros((tokens - 70, 32)), torch.nn.functional.pad(xq, (0, 12))])[:, :cols]
    xs = torch.cat([torch.ones(tokens - 70, device="cuda"), xs])
    y = int8_linear(xq, xs, wq, ws)
    check_linear(y[-70:], product64(xq[-70:], xs[-70:], wq, ws))
    assert not bool(y[:-70].any())
    with pytest.raises(ValueError, match="tokens"):
        int8_linear(torch.zeros((tokens + 1, 16), dtype=torch.int8, device="cuda"),
                    torch.zeros(tokens + 1, device="cuda"), wq[:, :16], ws)
    del y
    both = product64(xq[-70:], xs[-70:], wq, ws)
    h = int8_gated_linear(xq, xs, wq, ws)
    check_gated(h[-70:], both[:, :rows // 2], both[:, rows // 2:])


def test_threads_share_norms_and_layers():
    """Two threads on streams of their own call one norm and one layer at the same time, eagerly and replaying graphs."""
    hidden, inner = 512, 1200
    gen = torch.Generator().manual_seed(0)

    def make(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen) * scale).to(BF16).cuda()

    norm = BlockNorm(1 + make(hidden, scale=0.1))
    ffn = Int8GatedFFN.from_weights(make(inner, hidden, scale=0.06), make(inner, hidden, scale=0.06),
                                    make(hidden, inner, scale=0.04))
    inputs = [make(t, hidden) for t in (3, 700)]

    def step(x):
        return residual_norm(ffn(norm(x, quantize=True), out_dtype=BF16), x, next_norm=norm)

    want = [step(x) for x in inputs]
    graphs, captured = [], []
    for x in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.append(step(x))
        graphs.append(graph)
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for k in range(30):
                r, x = step(inputs[i])
                graphs[i].replay()
                stream.synchronize()
                for got in ((r, x), captured[i]):
                    if not (torch.equal(got[0], want[i][0]) and torch.equal(got[1], want[i][1])):
                        wrong.append((i, k))
            stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not wrong
