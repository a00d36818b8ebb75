"""Block norms, the fused residual join and row quantisation against their formulas in float64.

Tolerance of a float output, per element: half a step of the output's type on
the value, plus 256 * 2^-24 of the row's largest magnitude (of the value or of
what is summed to it).  A thread adds at most 32 terms in turn and the block
10 levels of pairs, so a row sum is within 43 * 2^-24 of exact; its root
halves that, and the two norms with the products between them stay below
2 * (43 + 20) * 2^-24 of the largest term, doubled again for the second
norm's own statistics over perturbed values.
"""
from __future__ import annotations

import math

import pytest
import torch

import conftest  # noqa: F401
from qcc_b200.runtime.block_norm import BlockNorm, quantize_rows, residual_norm

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def norm64(v, norm):
    if norm is None:
        return v
    if norm.kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / (v.square().mean(-1, keepdim=True) + norm.eps).sqrt()
    if norm.weight is not None:
        v = v * (norm.weight.double() + norm.weight_offset)
    return v if norm.bias is None else v + norm.bias.double()


def assert_rows_close(got, want, extra=None):
    want = want.double()
    scale = want.abs().amax(-1, keepdim=True)
    if extra is not None:
        scale = torch.maximum(scale, extra.double().abs().amax(-1, keepdim=True))
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half * 2
    bound = half * want.abs() + 256 * U32 * scale + tiny
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


def make(shape, dtype, seed, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale + shift).to(dtype).cuda()


def make_norm(hidden, kind, dtype, seed, bias=True, offset=0.0, weight=True):
    w = make(hidden, dtype, seed, 0.2, 1.0 - offset) if weight else None
    b = make(hidden, dtype, seed + 1, 0.2) if bias else None
    return BlockNorm(w, b, kind=kind, weight_offset=offset)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (1, 7), (3, 8), (2, 33), (5, 64), (4, 1111), (1, 5120), (9, 5120),
                                         (300, 256), (2, 4104), (2, 8191), (3, 17408), (1, 32768), (2, 32767)])
def test_norm_matches_formula(rows, hidden, kind, dtype):
    x = make((rows, hidden), dtype, 3, 2.0, 0.5)
    norm = make_norm(hidden, kind, dtype, 5)
    y = norm(x)
    assert y.dtype == dtype and y.shape == x.shape
    assert_rows_close(y, norm64(x.double(), norm), norm.bias.expand(rows, hidden))


@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("param_dtype", DTYPES)
def test_norm_types_and_offset(param_dtype, out_dtype):
    x = make((6, 520), torch.bfloat16, 1)
    norm = make_norm(520, "rms", param_dtype, 2, bias=False, offset=1.0)
    assert_rows_close(norm(x, out_dtype=out_dtype), norm64(x.double(), norm))
    bare = BlockNorm(kind="layer", eps=1e-5)
    assert_rows_close(bare(x, out_dtype=out_dtype), norm64(x.double(), bare))


@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hidden", [(1, 64), (5, 333), (3, 1000), (2, 5120), (700, 1111), (9, 20001)])
def test_fp32_rows_for_16_bit_weights(rows, hidden, low):
    """An fp32 residual stream normed with 16-bit parameters, into 16 bits, fp32 and int8."""
    x = make((rows, hidden), torch.float32, 1, 2.0)
    for kind, param_dtype in (("rms", low), ("layer", low), ("layer", torch.float32)):
        norm = make_norm(hidden, kind, param_dtype, 2)
        want = norm64(x.double(), norm)
        for out_dtype in (low, torch.float32):
            y = norm(x, out_dtype=out_dtype)
            assert y.dtype == out_dtype
            assert_rows_close(y, want, norm.bias.expand(rows, hidden))
        q, s = norm(x, quantize=True)
        amax = want.abs().amax(-1, keepdim=True)
        bound = 260 * U32 * (amax + norm.bias.double().abs().max())
        assert bool(((s.double()[:, None] * 127 - amax).abs() <= bound).all())
        assert bool(((q.double() * s.double()[:, None] - want).abs() <= 0.5 * amax / 127 + 127 * 4 * U32 * amax
                     + 2 * bound).all())


def test_norm_strides_views_and_in_place():
    base = make((7, 1300), torch.bfloat16, 4)
    norm = make_norm(640, "rms", torch.bfloat16, 5, bias=False)
    for x in (base[:, 16:656], base[:, 3:643], base[::2, :640], base[:1, 1:641], base[:, 640].expand(640, 7).t()):
        assert_rows_close(norm(x), norm64(x.double(), norm))
    x = make((2, 5, 640), torch.bfloat16, 6)
    assert_rows_close(norm(x).view(10, 640), norm64(x.double(), norm).view(10, 640))
    row = make((640,), torch.bfloat16, 7)
    assert norm(row).shape == (640,)
    assert torch.equal(norm(row), norm(row[None])[0])
    expanded = row.expand(4, 640)
    assert torch.equal(norm(expanded), norm(row[None]).expand(4, 640))
    want = norm(x)
    assert norm(x, out=x) is x and torch.equal(x, want)
    wide = torch.full((3, 700), 9.0, dtype=torch.bfloat16, device="cuda")
    x = make((3, 640), torch.bfloat16, 8)
    norm(x, out=wide[:, :640])
    assert torch.equal(wide[:, :640], norm(x)) and bool((wide[:, 640:] == 9).all())


@pytest.mark.parametrize("hidden", [100, 1111, 2049, 5120])
@pytest.mark.parametrize("rows", [1, 2, 7, 700])
@pytest.mark.parametrize("offsets,pads", [((3, 3, 3, 3), (5, 5, 5, 5)), ((0, 0, 0, 0), (3, 11, 3, 19)),
                                          ((1, 9, 1, 17), (0, 0, 0, 0)), ((0, 1, 2, 3), (8, 7, 6, 5))])
def test_join_of_views_writes_nothing_else(hidden, rows, offsets, pads):
    """Branch, residual and outputs as views into wider buffers, their rows sharing 16-byte granules or not."""
    buffers, views = [], []
    for i, (offset, pad) in enumerate(zip(offsets, pads)):
        flat = make((offset + rows * (hidden + pad) + 16,), torch.bfloat16, 20 + i)
        buffers.append(flat)
        views.append(flat.as_strided((rows, hidden), (hidden + pad, 1), offset))
    branch, residual, r_out, x_out = views
    norm = make_norm(hidden, "layer", torch.bfloat16, 30)
    gate = make((rows, hidden + 3), torch.bfloat16, 33)[:, 1:hidden + 1]
    want = residual_norm(branch.contiguous(), residual.contiguous(), post=norm, gate=gate.contiguous(), next_norm=norm)
    kept = [b.clone() for b in buffers]
    r, x = residual_norm(branch, residual, post=norm, gate=gate, next_norm=norm, residual_out=r_out, out=x_out)
    assert r is r_out and x is x_out
    for got, expected, b in ((r, want[0], None), (x, want[1], None)):
        scale = expected.double().abs().amax(-1, keepdim=True) + 4  # sums in another order: 256 roundings, one step
        assert bool(((got.double() - expected.double()).abs()
                     <= torch.finfo(got.dtype).eps * expected.double().abs() + 512 * U32 * scale).all())
    for i, (now, before) in enumerate(zip(buffers, kept)):
        if i >= 2:
            now.as_strided((rows, hidden), (hidden + pads[i], 1), offsets[i]).zero_()
            before.as_strided((rows, hidden), (hidden + pads[i], 1), offsets[i]).zero_()
        assert torch.equal(now, before)
    # The same in place, over the branch and the residual.
    r, x = residual_norm(branch, residual, post=norm, gate=gate, next_norm=norm, residual_out=residual, out=branch)
    assert bool(((x.double() - want[1].double()).abs() <= torch.finfo(x.dtype).eps * want[1].double().abs()
                 + 512 * U32 * (want[1].double().abs().amax(-1, keepdim=True) + 4)).all())


def test_norm_extremes():
    norm = BlockNorm(kind="rms", eps=1e-6)
    x = torch.zeros((6, 100), device="cuda")
    x[1] = 1e-30
    x[2] = 1e18
    x[3, 5] = float("nan")
    x[4, 5] = float("inf")
    y = norm(x)
    assert bool((y[0] == 0).all()) and bool((y[1] == 1e-30 * 1000).logical_or((y[1] - 1e-27).abs() < 1e-33).all())
    assert torch.allclose(y[2], torch.ones_like(y[2]), rtol=1e-6)
    assert bool(y[3].isnan().all()) and bool(y[4, 5].isnan())
    assert bool((y[5] == 0).all())
    assert norm(x[:0]).shape == (0, 100)
    q, s = norm(x[:0], quantize=True)
    assert q.shape == (0, 100) and s.shape == (0,)


GATES = [None, "token", "channel", "full", "scalar"]


@pytest.mark.parametrize("dtype,res_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                             (torch.float16, torch.float16), (torch.float16, torch.float32),
                                             (torch.float32, torch.float32)])
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("rows,hidden", [(1, 5120), (3, 1111), (65, 256), (2, 9000), (2, 20000), (1, 32768)])
def test_join_matches_formula(rows, hidden, gate, dtype, res_dtype):
    branch, residual = make((rows, hidden), dtype, 1), make((rows, hidden), res_dtype, 2, 3.0)
    shape = {None: None, "token": (rows, 1), "channel": (hidden,), "full": (rows, hidden), "scalar": (1,)}[gate]
    g = None if shape is None else make(shape, dtype, 3)
    post, following = make_norm(hidden, "rms", dtype, 4), make_norm(hidden, "layer", torch.float32, 6)
    act = {"token": "sigmoid", "channel": "tanh"}.get(gate)
    r, x = residual_norm(branch, residual, post=post, gate=g, gate_activation=act, residual_scale=0.75,
                         branch_scale=-1.5, next_norm=following)
    b = norm64(branch.double(), post)
    if g is not None:
        g64 = g.double()
        b = b * (g64.sigmoid() if act == "sigmoid" else g64.tanh() if act == "tanh" else g64)
    want = 0.75 * residual.double() - 1.5 * b
    assert r.dtype == res_dtype and x.dtype == dtype
    assert_rows_close(r, want, 3 * torch.maximum(b.abs(), residual.double().abs()))
    following64 = norm64(want, following)
    assert_rows_close(x, following64, 4 * following64.abs() + following.bias.double().abs() + 4)
    # Without norms on either side the join is a scaled sum.
    alone = residual_norm(branch, residual, gate=g, branch_scale=0.5)
    b = branch.double() if g is None else branch.double() * g.double()
    assert_rows_close(alone, residual.double() + 0.5 * b, torch.maximum(b.abs(), residual.double().abs()))


def test_join_gate_of_sequences_and_in_place():
    branch, residual = make((2, 5, 64), torch.bfloat16, 1), make((2, 5, 64), torch.bfloat16, 2)
    for shape in ((2, 1, 64), (2, 1, 1), (1, 1, 64), (64,), (2, 5, 1), (2, 5, 64), (5, 1), (1, 5, 64)):
        g = make(shape, torch.float32, 3)
        if shape in ((5, 1), (1, 5, 64)):  # shared along a leading axis only: not a run of consecutive rows
            with pytest.raises(ValueError, match="broadcast"):
                residual_norm(branch, residual, gate=g)
            continue
        r = residual_norm(branch, residual, gate=g)
        b = branch.double() * g.double()
        assert_rows_close(r.view(10, 64), (residual.double() + b).view(10, 64), b.view(10, 64))
    norm = make_norm(64, "rms", torch.bfloat16, 4)
    want = residual_norm(branch, residual, next_norm=norm)
    keep = branch.clone()
    r, x = residual_norm(branch, residual, next_norm=norm, residual_out=residual, out=branch)
    assert r is residual and x is branch
    assert torch.equal(r, want[0]) and torch.equal(x, want[1])
    # The fused norm sees the sum before its rounding; with an fp32 residual the two steps agree to fp32 (both are
    # within the bound of the exact value, with contractions of their own, so their bits may differ).
    res32 = make((2, 5, 64), torch.float32, 9)
    r, x = residual_norm(keep, res32, next_norm=norm, out_dtype=torch.float32)
    again = norm(r, out_dtype=torch.float32)
    assert_rows_close(x.view(10, 64), again.view(10, 64), again.view(10, 64))


def quantized_plain(v):
    """The documented rule.  In float64 127 v is exact and its quotient by amax rounds to a border (k + 1/2) only where
    it is one: another quotient of a 31-bit by a 24-bit number is at least 2^-25 away."""
    v = v.double().cpu()
    amax = v.abs().amax(-1, keepdim=True)
    keep = amax >= 2.0 ** -119
    q = torch.where(keep, torch.round(127 * v / amax), torch.zeros_like(v))
    return q.to(torch.int8), torch.where(keep, amax / 127, torch.zeros_like(amax)).float()[:, 0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 15), (3, 16), (5, 33), (64, 517), (2, 5120), (3, 17408), (1, 32768),
                                       (2, 30001)])
def test_quantize_rows(rows, cols, dtype):
    x = make((rows, cols), dtype, 11, 3.0)
    q, s = quantize_rows(x)
    assert q.shape == x.shape and q.stride(0) % 16 == 0 and q.data_ptr() % 16 == 0
    want_q, want_s = quantized_plain(x)
    assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)
    step = s.double()[:, None]
    assert bool(((q.double() * step - x.double()).abs() <= step * (0.5 + 127 * 4 * U32)).all())
    assert bool((q.abs().amax(1) == 127).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows_on_borders(dtype):
    """Rows full of values on or next to a border between two steps, at ordinary, tiny and huge magnitudes."""
    cols = 2 * 127 + 2
    for amax in (254.0, 127.0, 3 * 127.0, 1.0, 0.7, 254 * 2.0 ** -20, 254 * 2.0 ** -60, 2.0 ** 127 * 1.984):
        if dtype == torch.float16 and not 2.0 ** -14 <= amax < 65504:
            continue
        a = float(torch.tensor(amax).to(dtype))
        steps = torch.arange(-127, 127, dtype=torch.float64) + 0.5
        x = torch.cat([steps * a / 127, torch.tensor([a, -a], dtype=torch.float64)]).to(dtype)
        bits = x.float().view(torch.int32)
        unit = 1 if dtype == torch.float32 else 1 << (16 if dtype == torch.bfloat16 else 13)
        rows = [x]
        for shift in (-unit, unit):  # the neighbours of each value in its type, kept below amax
            rows.append(torch.where(x.float().abs() < a, (bits + shift).view(torch.float32), x.float()).to(dtype))
        x = torch.stack(rows).cuda()
        assert x.shape[1] == cols
        for y in (x, x[:, :cols - 1].flip(1)):  # with and without the granule kernels' alignment
            q, s = quantize_rows(y.contiguous())
            want_q, want_s = quantized_plain(y)
            assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s), amax
        q, s = quantize_rows(x.contiguous().view(-1)[3:3 + cols].view(1, cols))
        want_q, want_s = quantized_plain(x.contiguous().view(-1)[3:3 + cols].view(1, cols))
        assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_rows_over_a_whole_type(dtype):
    """Every value of the type up to amax, for a few amax of each significand's parity."""
    positive = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16).view(dtype).float()
    for amax in (1.0, 1.5, 1.0078125, 1.9921875, 240.0, 1.25 * 2.0 ** -10, 127.0, 0.99609375):
        x = positive[positive <= amax].to(dtype)
        assert float(x.float().max()) == amax
        for y in (x, -x):
            q, s = quantize_rows(y.cuda()[None])
            want_q, want_s = quantized_plain(y[None])
            assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s), amax


def test_quantize_rows_extremes():
    x = torch.zeros((8, 40), device="cuda")
    x[1] = 2.0 ** -119
    x[2] = 2.0 ** -120
    x[3, 1] = float("nan")
    x[4, 2] = float("-inf")
    x[5] = 3e38
    x[6, 0], x[6, 1] = -1.0, 0.5
    q, s = quantize_rows(x)
    assert s[0] == 0 and bool((q[0] == 0).all())
    assert s[1] > 0 and bool((q[1] == 127).all())
    assert s[2] == 0 and bool((q[2] == 0).all())
    for row in (3, 4):
        assert s[row].isnan() and bool((q[row] == 0).all())
    assert s[5].isfinite() and bool((q[5] == 127).all())
    assert q[6, 0] == -127 and q[6, 1] == 64  # 63.5 to the even side
    assert bool((q[7] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,hidden", [(1, 5120), (7, 517), (33, 512)])
def test_norm_quantized(rows, hidden, dtype):
    """int8 rows of the norm: within half a step, plus what the fp32 norm is off, of the norm in float64."""
    x, residual = make((rows, hidden), dtype, 1), make((rows, hidden), dtype, 2)
    norm = make_norm(hidden, "rms", dtype, 3)
    for q, s, want in ((*norm(x, quantize=True), norm64(x.double(), norm)),
                       (*residual_norm(x, residual, next_norm=norm, quantize=True)[1],
                        norm64(x.double() + residual.double(), norm))):
        amax = want.abs().amax(-1, keepdim=True)
        assert bool(((s.double()[:, None] * 127 - amax).abs() <= 260 * U32 * amax).all())
        assert bool(((q.double() * s.double()[:, None] - want).abs()
                     <= 0.5 * amax / 127 + (260 + 127 * 4) * U32 * amax).all())


@pytest.mark.parametrize("hidden", [8, 100, 1111, 5120])
def test_norm_quantized_extremes(hidden):
    x = make((5, hidden), torch.float32, 1)
    x[1, hidden // 2] = float("nan")
    x[2, 0] = float("inf")
    x[3] = 0
    for norm in (make_norm(hidden, "rms", torch.float32, 2, bias=False), make_norm(hidden, "layer", torch.float32, 3)):
        q, s = norm(x, quantize=True)
        assert bool(s[1:3].isnan().all()) and bool((q[1:3] == 0).all())
        assert bool(s[[0, 4]].isfinite().all())
        if norm.bias is None:
            assert s[3] == 0 and bool((q[3] == 0).all())


def test_replaced_parameters():
    """A norm follows its parameters when a module replaces their data, and refuses what no longer fits."""
    x = make((5, 512), torch.float32, 1)
    weight, bias = make((512,), torch.float32, 2), make((512,), torch.float32, 3)
    layer = torch.nn.LayerNorm(512, device="cuda").requires_grad_(False)
    layer.weight.data, layer.bias.data = weight.clone(), bias.clone()
    norm = BlockNorm(layer.weight, layer.bias, kind="layer")
    assert torch.equal(norm(x), BlockNorm(weight, bias, kind="layer")(x))
    layer.half()
    assert torch.equal(norm(x), BlockNorm(weight.half(), bias.half(), kind="layer")(x))
    layer.float()
    layer.weight.data = layer.weight.data[:100]  # the same address, fewer values
    with pytest.raises(ValueError):
        norm(x)
    layer.bias.data = layer.bias.data[:100]
    with pytest.raises(ValueError):
        norm(x)
    assert torch.equal(norm(x[:, :100]), BlockNorm(layer.weight, layer.bias, kind="layer")(x[:, :100]))
    layer.weight.data = torch.ones(200, device="cuda")[::2]
    with pytest.raises(ValueError):
        norm(x[:, :100])
    layer.weight.data = torch.ones(100, device="cuda", dtype=torch.float16)
    with pytest.raises(TypeError):
        norm(x[:, :100])
    layer.cpu()
    with pytest.raises(RuntimeError):
        norm(x[:, :100])


def test_streams_and_graph():
    x, residual = make((9, 5120), torch.bfloat16, 1), make((9, 5120), torch.bfloat16, 2)
    norm = make_norm(5120, "rms", torch.bfloat16, 3)
    want = residual_norm(x, residual, post=norm, next_norm=norm)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = residual_norm(x, residual, post=norm, next_norm=norm)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = residual_norm(x, residual, post=norm, next_norm=norm)
    x.copy_(make((9, 5120), torch.bfloat16, 8))
    want = residual_norm(x, residual, post=norm, next_norm=norm)
    graph.replay()
    assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1])


@pytest.mark.parametrize("rows,hidden", [(2048, 1400), (2049, 1536), (2051, 2048), (2048, 1401)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_of_middling_width(rows, hidden, dtype):
    x, residual = make((rows, hidden), dtype, 1), make((rows, hidden), dtype, 2)
    norm = make_norm(hidden, "layer", dtype, 3)
    assert_rows_close(norm(x), norm64(x.double(), norm), norm.bias.expand(rows, hidden))
    bare = make_norm(hidden, "rms", dtype, 5, bias=False)
    r, (q, s) = residual_norm(x, residual, next_norm=bare, quantize=True)
    want = x.double() + residual.double()
    assert_rows_close(r, want, torch.maximum(x.abs(), residual.abs()))
    want = norm64(want, bare)
    amax = want.abs().amax(-1, keepdim=True)
    assert bool(((q.double() * s.double()[:, None] - want).abs() <= 0.5 * amax / 127 + (520 + 127 * 4) * U32 * amax).all())
    q, s = quantize_rows(x)
    want_q, want_s = quantized_plain(x)
    assert torch.equal(q.cpu(), want_q) and torch.equal(s.cpu(), want_s)


def test_many_rows():
    """More rows than one launch dimension of 65535 would hold."""
    rows = 70001
    x = make((rows, 16), torch.float16, 1)
    norm = BlockNorm(kind="rms")
    assert_rows_close(norm(x), norm64(x.double(), norm))
    assert math.isclose(float(norm(x)[-1].double().square().mean()), 1.0, rel_tol=1e-2)
