"""8-bit integer products against their formula in float64, and the layer built from them.

Tolerances: the integer sums are exact (float64 holds them), so an output is
off by half a step of its type, plus the fp32 roundings of the sum's
conversion, the scales' product, their product and the bias (4 * 2^-24 of the
terms).  The gated form: g and u carry 3 roundings each, their product 1; of
silu's, exp is off by 2 ulp (4 roundings), the sum by 1, the quotient by 2 ulp,
16 in all; and exp turns the 3 roundings of g, with 1 of its own argument's
scaling, into 4 |g|.  Below g = -87.3 the quotient becomes 0: an error of its
value, less than |g| exp(g) |u|, which 2^-119 |u| bounds.
"""
from __future__ import annotations

import pytest
import torch

import conftest  # noqa: F401
from qcc_b200.runtime.block_norm import BlockNorm, int8_rows, quantize_rows, residual_norm
from qcc_b200.runtime.int8_dense import (Int8GatedFFN, Int8GatedLinear, Int8Linear, int8_gated_linear, int8_linear)

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def int8_matrix(rows, cols, seed, low=-128, high=127):
    gen = torch.Generator().manual_seed(seed)
    whole = torch.randint(-128, 128, (rows, (cols + 15) // 16 * 16), generator=gen, dtype=torch.int8)
    whole[:, :cols] = torch.randint(low, high + 1, (rows, cols), generator=gen, dtype=torch.int8)
    return whole.cuda()[:, :cols]  # the padding holds values


def scales(n, seed, size=1.0):
    gen = torch.Generator().manual_seed(seed)
    return ((0.5 + torch.rand(n, generator=gen)) * size).cuda()


def operands(tokens, rows, cols, seed=0):
    size = 1 / (74 * 74 * cols ** 0.5)
    return (int8_matrix(tokens, cols, seed), scales(tokens, seed + 1), int8_matrix(rows, cols, seed + 2),
            scales(rows, seed + 3, size))


def product64(xq, xs, wq, ws):
    return (xq.double() @ wq.double().t()) * xs.double()[:, None] * ws.double()


def check_linear(y, want, bias=None):
    terms = want.abs() + (0 if bias is None else bias.double().abs())
    want = want if bias is None else want + bias.double()
    half = torch.finfo(y.dtype).eps / 2
    tiny = torch.finfo(y.dtype).smallest_normal * half * 2
    off = (y.double() - want).abs()
    bound = half * want.abs() + 4 * U32 * terms * (1 + half) + tiny
    assert bool((off <= bound).all()), float((off / bound).max())


def check_gated(h, g, u):
    want = g * torch.sigmoid(g) * u
    half = torch.finfo(h.dtype).eps / 2
    tiny = torch.finfo(h.dtype).smallest_normal * half * 2
    off = (h.double() - want).abs()
    bound = want.abs() * (half + (16 + 4 * g.abs()) * U32 * 1.01) + tiny + 2.0 ** -119 * u.abs()
    assert bool((off <= bound).all()), float((off / bound).max())


SHAPES = [(1, 1, 1), (1, 5, 16), (2, 16, 15), (3, 129, 33), (1, 256, 5120), (8, 130, 517), (16, 64, 64), (17, 65, 129),
          (33, 1000, 1111), (64, 127, 128), (65, 255, 2048), (127, 300, 640), (128, 128, 128), (129, 257, 255),
          (255, 512, 384), (257, 513, 1025), (300, 1023, 517), (513, 640, 1280), (1000, 384, 100), (2, 5120, 17408),
          (1, 17408, 5120), (1025, 1500, 2000)]


@pytest.mark.parametrize("tokens,rows,cols", SHAPES)
def test_linear_matches_formula(tokens, rows, cols):
    xq, xs, wq, ws = operands(tokens, rows, cols)
    want = product64(xq, xs, wq, ws)
    gen = torch.Generator().manual_seed(9)
    for dtype in DTYPES:
        check_linear(int8_linear(xq, xs, wq, ws, out_dtype=dtype), want)
        bias = torch.randn(rows, generator=gen).to(dtype).cuda()
        check_linear(int8_linear(xq, xs, wq, ws, bias=bias, out_dtype=dtype), want, bias)


@pytest.mark.parametrize("tokens,rows,cols", SHAPES)
def test_gated_matches_formula(tokens, rows, cols):
    xq, xs, wq, ws = operands(tokens, 2 * rows, cols)
    both = product64(xq, xs, wq, ws)
    for dtype in DTYPES:
        check_gated(int8_gated_linear(xq, xs, wq, ws, out_dtype=dtype), both[:, :rows], both[:, rows:])


def test_default_output_is_bf16_and_out_buffers():
    xq, xs, wq, ws = operands(5, 70, 96)
    y = int8_linear(xq, xs, wq, ws)
    assert y.dtype == torch.bfloat16
    wide = torch.full((5, 99), 7.0, device="cuda")
    out = wide[:, 3:73]
    assert int8_linear(xq, xs, wq, ws, out=out) is out
    check_linear(out, product64(xq, xs, wq, ws))
    assert bool((wide[:, :3] == 7).all()) and bool((wide[:, 73:] == 7).all())


@pytest.mark.parametrize("tokens", [1, 2, 40, 256, 700])
def test_rows_beyond_the_output_are_left(tokens):
    xq, xs, wq, ws = operands(tokens, 2 * 133, 80)
    for gated, channels in ((False, 266), (True, 133)):
        for dtype in DTYPES:
            flat = torch.full((tokens * channels + 64,), 7.0, dtype=dtype, device="cuda")
            out = flat[:tokens * channels].view(tokens, channels)
            (int8_gated_linear if gated else int8_linear)(xq, xs, wq, ws, out=out)
            assert bool((flat[tokens * channels:] == 7).all())


def test_extreme_values():
    """The largest sums (every product 128 * 128, and 127 * -128) at the largest column count, and odd scales."""
    cols = 131071
    xq, wq = int8_rows(3, cols, torch.device("cuda")), int8_rows(4, cols, torch.device("cuda"))
    xq[:], wq[:] = -128, -128
    xq[1], wq[2:] = 127, 127
    xs = torch.tensor([1.0, 1.0, 0.0], device="cuda")
    ws = torch.tensor([1.0, 2.0 ** -126, 1.0, float("nan")], device="cuda")
    y = int8_linear(xq, xs, wq, ws, out_dtype=torch.float32)
    want = (xq.double() @ wq.double().t())
    assert torch.equal(y[:2, 0].double(), want[:2, 0].float().double())
    assert torch.equal(y[:2, 2].double(), want[:2, 2].float().double())
    assert float(y[0, 1]) == float(want[0, 1].float()) * 2.0 ** -126
    assert bool((y[2, :3] == 0).all()) and bool(y[:, 3].isnan().all())
    # g far below zero: silu and its product go to zero, not to NaN.
    h = int8_gated_linear(xq[1:2], torch.ones(1, device="cuda"), wq[0::2],
                          torch.ones(2, device="cuda"), out_dtype=torch.float32)
    assert float(h) == 0.0


def test_no_tokens():
    xq, xs, wq, ws = operands(0, 64, 32)
    assert int8_linear(xq, xs, wq, ws).shape == (0, 64)
    assert int8_gated_linear(xq, xs, wq, ws).shape == (0, 32)


def test_repeated_calls_agree_bit_for_bit():
    xq, xs, wq, ws = operands(37, 1000, 4000)
    first = int8_linear(xq, xs, wq, ws)
    for _ in range(3):
        assert torch.equal(int8_linear(xq, xs, wq, ws), first)
    # A token's result does not depend on the batch it comes in (integer sums, the same fp32 steps).
    for t in (1, 5, 17):
        assert torch.equal(int8_linear(xq[:t], xs[:t], wq, ws), first[:t])


def test_streams_and_graphs_run_side_by_side():
    """Two graphs captured on one stream and replayed on two, and eager calls beside them."""
    a, b = operands(4, 512, 8192, 0), operands(4, 512, 8192, 50)
    want_a, want_b = int8_linear(*a), int8_gated_linear(*b)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        got_a = int8_linear(*a)
    with torch.cuda.graph(graphs[1]):
        got_b = int8_gated_linear(*b)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        got_a.zero_()
        got_b.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = int8_linear(*a)
        torch.cuda.synchronize()
        assert torch.equal(got_a, want_a) and torch.equal(got_b, want_b) and torch.equal(eager, want_a)


def test_linear_classes():
    gen = torch.Generator().manual_seed(0)
    w = torch.randn(96, 72, generator=gen).bfloat16().cuda()
    x = torch.randn(2, 3, 72, generator=gen).bfloat16().cuda()
    bias = torch.randn(96, generator=gen).bfloat16().cuda()
    layer = Int8Linear.from_weight(w, bias)
    y = layer(x)
    assert y.shape == (2, 3, 96) and y.dtype == torch.bfloat16
    xq, xs = quantize_rows(x)
    assert torch.equal(y.view(6, 96), int8_linear(xq, xs, layer.weight, layer.scale, bias=bias))
    assert torch.equal(layer((xq, xs)), y.view(6, 96))
    exact = x.double().view(6, 72) @ w.double().t() + bias.double()
    # Each operand is off by half a step, amax / 254: an entry's errors add up over 72 columns.
    xa, wa = x.double().view(6, 72).abs(), w.double().abs()
    bound = (xa.amax(1)[:, None] / 254) * wa.sum(1) + xa.sum(1)[:, None] * wa.amax(1) / 254 \
        + 72 * xa.amax(1)[:, None] * wa.amax(1) / 254 ** 2 + 2.0 ** -8 * (exact.abs() + 1)
    assert bool(((y.view(6, 96).double() - exact).abs() <= bound).all())
    gated = Int8GatedLinear.from_weights(w[:48], w[48:])
    whole = Int8GatedLinear.from_weight(w)
    assert torch.equal(gated.weight, whole.weight) and torch.equal(gated.scale, whole.scale)
    assert torch.equal(gated(x), whole(x)) and gated(x).shape == (2, 3, 48)
    one = torch.randn(72, generator=gen).bfloat16().cuda()
    assert layer(one).shape == (96,)


@pytest.mark.parametrize("tokens", [1, 5, 130])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_run_together(tokens, dtype):
    """residual -> norm (int8) -> gate | up -> int8 -> down -> norm, gate and sum -> next norm, against float64."""
    hidden, inner = 264, 520
    gen = torch.Generator().manual_seed(1)

    def make(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen) * scale).to(dtype).cuda()

    gate, up, down = make(inner, hidden, scale=0.06), make(inner, hidden, scale=0.06), make(hidden, inner, scale=0.04)
    residual, token_gate = make(tokens, hidden, scale=2.0), make(tokens, 1)
    pre, post, following = (BlockNorm((1 + make(hidden, scale=0.1)).contiguous()) for _ in range(3))
    ffn = Int8GatedFFN.from_weights(gate, up, down)
    assert ffn.hidden == hidden and ffn.intermediate == inner
    q, s = pre(residual, quantize=True)
    y = ffn((q, s), out_dtype=dtype)
    r, x = residual_norm(y, residual, post=post, gate=token_gate, gate_activation="sigmoid", next_norm=following)

    # float64, with the operands' quantised values and the stored activation's rounding.
    both = product64(q, s, ffn.gate_up.weight, ffn.gate_up.scale)
    h = torch.nn.functional.silu(both[:, :inner]) * both[:, inner:]
    stored = ffn.gate_up((q, s), out_dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16)
    check_gated(stored, both[:, :inner], both[:, inner:])
    assert stored.shape == h.shape
    hq, hs = quantize_rows(stored)
    y64 = product64(hq, hs, ffn.down.weight, ffn.down.scale)
    check_linear(y, y64)

    def rms(v, norm):
        return v / (v.square().mean(-1, keepdim=True) + norm.eps).sqrt() * norm.weight.double()

    branch = token_gate.double().sigmoid() * rms(y.double(), post)
    want = residual.double() + branch
    half = torch.finfo(dtype).eps / 2
    scale = want.abs().amax(1, keepdim=True) + branch.abs().amax(1, keepdim=True)
    assert bool(((r.double() - want).abs() <= half * want.abs() + 256 * U32 * scale).all())
    want_x = rms(want, following)
    assert bool(((x.double() - want_x).abs()
                 <= half * want_x.abs() + 1024 * U32 * want_x.abs().amax(1, keepdim=True)).all())

    # The whole layer is near the dense layer in float64: int8's errors, about 1% each in the 2-norm.
    n = rms(residual.double(), pre)
    dense = (torch.nn.functional.silu(n @ gate.double().t()) * (n @ up.double().t())) @ down.double().t()
    assert float((y.double() - dense).norm() / dense.norm()) < 0.05
