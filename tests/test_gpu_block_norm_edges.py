"""Block norms, the join and row quantisation where they can go wrong: borders of the int8 form, waits that run out."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import conftest  # noqa: F401
from qcc_b200 import _lib
from qcc_b200.runtime.block_norm import BlockNorm, quantize_rows, residual_norm
from qcc_b200.runtime.int8_dense import int8_gated_linear, int8_linear
from test_gpu_block_norm import assert_rows_close, norm64

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def make(shape, dtype, seed, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale + shift).to(dtype).cuda()


def int8_of_products(u):
    """round_half_even of 127 u / amax in fp32, for fp32 products u.  In float64 127 u is exact, and its quotient's
    rounding to float64 moves it over no border between two fp32 numbers: a quotient of a 31-bit by a 24-bit number
    that is no such border is 2^-49 or more of itself away from one."""
    u = u.double()
    amax = u.abs().amax(-1, keepdim=True)
    return torch.round((127 * u / amax).float()).to(torch.int8), amax


def rows_with_ties(rows, hidden, dtype, weight_dtype, seed):
    """Rows and weights whose products are half of the largest one in many places, by factors of other significands."""
    x = make((rows, hidden), dtype, seed, 0.3).clamp(-1.5, 1.5)
    w = make(hidden, weight_dtype, seed + 1, 0.1, 1.0).clamp(0.5, 1.5)
    big_x = (3.0 + 0.5 * torch.rand(rows, 1, generator=torch.Generator().manual_seed(seed + 2))).to(BF16)
    big_w = 1.2109375
    x[:, hidden // 3] = big_x[:, 0].to(dtype).cuda()
    w[hidden // 3] = big_w
    ties = torch.arange(0, hidden, 7, device="cuda")
    ties = ties[ties != hidden // 3]
    half, same = ties[::2], ties[1::2]
    x[:, half], w[half] = (big_x / 2).to(dtype).cuda(), big_w       # half the value, the same weight
    x[:, same], w[same] = (big_x / 4).to(dtype).cuda().neg(), 2 * big_w
    return x, w


# Rows of a warp, of many warps, of the ring (refilled at 2200 x 2056 and 1300 x 4001), and of the kernel of single
# elements (16-bit rows with weights of the other 16-bit type).
@pytest.mark.parametrize("rows,hidden", [(3, 40), (5, 517), (9, 1000), (2049, 1536), (6, 5120), (2200, 2056),
                                         (1300, 4001), (2, 20000)])
@pytest.mark.parametrize("dtype,weight_dtype", [(BF16, BF16), (BF16, FP32), (FP16, FP16), (FP32, BF16), (FP32, FP32),
                                                (BF16, FP16), (FP16, BF16)])
def test_int8_of_an_rms_norm_rounds_the_products_quotient(rows, hidden, dtype, weight_dtype):
    x, w = rows_with_ties(rows, hidden, dtype, weight_dtype, 3)
    for offset in (0.0, 1.0):
        weight = (w.float() - offset).to(weight_dtype)
        norm = BlockNorm(weight, weight_offset=offset)
        u = x.float() * (weight.float() + offset)
        want, amax = int8_of_products(u)
        q, s = norm(x, quantize=True)
        assert torch.equal(q, want)
        # The scale: the mean of squares is within 43 * 2^-24 of exact (its root halves that), and rsqrt, the product,
        # the quotient and the factor round 6 times.
        size = (x.double().square().mean(1, keepdim=True) + norm.eps).sqrt()
        exact = amax / size / 127
        assert bool(((s.double()[:, None] - exact).abs() <= (22 + 6) * U32 * exact).all())
        if offset == 0.0 and dtype == weight_dtype:
            # Behind a join: the sum of branch and residual, rounded to fp32, takes the rows' place.
            residual = make((rows, hidden), dtype, 9, 0.25)
            want, _ = int8_of_products((x.float() + residual.float()) * weight.float())
            r, (q, s) = residual_norm(x, residual, next_norm=norm, quantize=True)
            assert torch.equal(q, want)


def test_int8_of_an_rms_norm_without_a_weight():
    x = make((7, 3000), BF16, 1)
    x[:, 5] = 8.0
    x[:, 9] = -4.0
    q, s = BlockNorm()(x, quantize=True)
    want, amax = int8_of_products(x.float())
    assert torch.equal(q, want) and bool((q[:, 9] == -64).all())


@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_int8_of_an_rms_norm_of_tiny_and_huge_rows(eps):
    """The row factor is a power of two and a rest: rows near fp32's ends keep their ratios and their scales."""
    base = make((6, 520), FP32, 4)
    x = base * torch.tensor([2.0 ** -60, 2.0 ** -58, 1.0, 2.0 ** 50, 2.0 ** 58, 0.0], device="cuda")[:, None]
    w = make(520, FP32, 5, 0.2, 1.0)
    q, s = BlockNorm(w, eps=eps)(x, quantize=True)
    want, amax = int8_of_products(x * w)
    assert torch.equal(q[:5], want[:5])
    exact = amax / (x.double().square().mean(1, keepdim=True) + eps).sqrt() / 127
    # Squares that fall below 2^-126 are off by 2^-150 each, 2^-36 of a row's sum of 2^-112 or more.
    assert bool(((s[:5].double()[:, None] - exact[:5]).abs() <= 28 * U32 * exact[:5]).all())
    assert bool(s[5].isnan()) if eps == 0.0 else float(s[5]) == 0.0
    assert bool((q[5] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows,cols", [(3, 32769), (5, 36864), (2, 53248), (1, 131071)])
def test_quantize_rows_as_wide_as_the_products(rows, cols, dtype):
    x = make((rows, cols), dtype, 4, 3.0)
    q, s = quantize_rows(x)
    amax = x.double().abs().amax(1, keepdim=True)
    want = torch.round(127 * x.double() / amax)  # exact but for borders, which are borders in float64 as well
    assert q.stride(0) % 16 == 0 and torch.equal(q.double(), want)
    assert torch.equal(s.cpu(), (amax[:, 0].cpu() / 127).float())
    with pytest.raises(ValueError, match="131071"):
        quantize_rows(torch.zeros((1, 131072), dtype=dtype, device="cuda"))
    with pytest.raises(ValueError, match="32768"):
        BlockNorm()(x, quantize=True)


def test_parameters_taken_away():
    """A norm whose weight or bias becomes None no longer reads the tensor that it had."""
    x = make((5, 512), FP32, 1)
    weight, bias = make(512, FP32, 2), make(512, FP32, 3)
    norm = BlockNorm(weight, bias, kind="layer")
    norm(x)
    norm.weight = None
    assert torch.equal(norm(x), BlockNorm(None, bias, kind="layer")(x))
    norm.bias = None
    assert norm.hidden is None and torch.equal(norm(x), BlockNorm(kind="layer")(x))
    assert torch.equal(norm(x[:, :100]), BlockNorm(kind="layer")(x[:, :100]))
    norm.weight, norm.bias = weight, bias
    assert norm.hidden == 512 and torch.equal(norm(x), BlockNorm(weight, bias, kind="layer")(x))
    shifted = BlockNorm(weight, weight_offset=1.0)
    shifted.weight = None
    with pytest.raises(ValueError, match="weight_offset"):
        shifted(x)


def test_tangents_are_refused():
    """A dual tensor's tangent would be dropped: the call is refused, and calls without one inside the level are not."""
    x, weight, gate = make((4, 64), FP32, 1), make(64, FP32, 2), make((4, 1), FP32, 3)
    norm = BlockNorm(weight)
    wq, ws = quantize_rows(make((8, 64), FP32, 4))
    xq, xs = quantize_rows(x)
    bias = make(8, FP32, 5)
    want = norm(x)
    with forward_ad.dual_level():
        dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, weight, gate, xs, ws, bias)]
        dual_x, dual_weight, dual_gate, dual_xs, dual_ws, dual_bias = dual
        for call in (lambda: norm(dual_x), lambda: norm(dual_x, quantize=True), lambda: quantize_rows(dual_x),
                     lambda: BlockNorm(dual_weight)(x), lambda: BlockNorm(weight, dual_weight)(x),
                     lambda: residual_norm(dual_x, x), lambda: residual_norm(x, dual_x),
                     lambda: residual_norm(x, x, gate=dual_gate),
                     lambda: residual_norm(x, x, post=BlockNorm(dual_weight)),
                     lambda: int8_linear(xq, dual_xs, wq, ws), lambda: int8_linear(xq, xs, wq, dual_ws),
                     lambda: int8_linear(xq, xs, wq, ws, bias=dual_bias),
                     lambda: int8_gated_linear(xq, dual_xs, wq, ws)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert torch.equal(norm(x), want)
        assert torch.equal(norm(forward_ad.unpack_dual(dual_x).primal), want)
    grad = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="quantize_rows has no backward"):
        quantize_rows(grad)
    with pytest.raises(RuntimeError):
        torch.func.jvp(norm, (x,), (x,))


@pytest.mark.parametrize("shape", [(64, 1), (64, 40), (64, 1029)])
def test_sigmoid_gate_far_from_zero(shape):
    """The sigmoid keeps its value down to fp32's smallest numbers, and large branches show it."""
    rows, cols = shape
    values = torch.cat([torch.linspace(-101.0, -80.0, 48), torch.tensor([-1e4, -float("inf"), float("inf"), 1e4, 0.0]),
                        torch.linspace(80.0, 101.0, 11)]).cuda()
    gate = values[:, None].expand(rows, cols).contiguous()
    hidden = max(cols, 40)
    branch = torch.full((rows, hidden), 1e30, device="cuda")
    r = residual_norm(branch, torch.zeros_like(branch), gate=gate, gate_activation="sigmoid")
    want = torch.sigmoid(gate.double()) * branch.double()
    # |g| + 8 roundings of the gate and one of the product; exp's smallest numbers are off by 2^-149 at most.
    bound = want * (values.double().abs().clamp(max=128.0)[:, None] + 10) * U32 + 2.0 ** -149 * branch.double()
    assert bool(((r.double() - want).abs() <= bound).all())
    assert bool((r[48] == 0).all()) and bool((r[49] == 0).all()) and bool((r[50] == branch[50]).all())


def close_int8(q, s, want, bound):
    """int8 rows of computed values: within half a step, and what the fp32 values are off (in their row's amax)."""
    amax = want.abs().amax(-1, keepdim=True)
    return bool(((q.double() * s.double()[:, None] - want).abs() <= 0.5 * amax / 127 + bound * U32 * amax).all())


# More rows a block than its ring holds, twice over: at 5120 values (16 bits) 592 to 1184 blocks of two or three rows.
@pytest.mark.parametrize("rows,hidden,dtype", [(6000, 5120, BF16), (6001, 4001, FP16), (4000, 5120, FP32),
                                               (3001, 2051, FP32), (2000, 12288, BF16), (1500, 20000, BF16)])
def test_rings_that_come_round(rows, hidden, dtype):
    x, residual = make((rows, hidden), dtype, 1, 2.0, 0.5), make((rows, hidden), dtype, 2)
    rms = BlockNorm(make(hidden, dtype, 3, 0.2, 1.0))
    layer = BlockNorm(make(hidden, dtype, 3, 0.2, 1.0), make(hidden, dtype, 4, 0.2), kind="layer")
    for norm in (rms, layer):
        want = norm64(x.double(), norm)
        extra = None if norm.bias is None else norm.bias.expand(rows, hidden)
        assert_rows_close(norm(x), want, extra)
        assert close_int8(*norm(x, quantize=True), want, 520 + 127 * 4)
    q, s = quantize_rows(x)
    amax = x.double().abs().amax(1, keepdim=True)
    assert torch.equal(q.double(), torch.round(127 * x.double() / amax))
    assert torch.equal(s, (amax[:, 0] / 127).float())
    b = norm64(x.double(), layer)
    want = residual.double() + 0.5 * b
    scale = torch.maximum(b.abs(), residual.double().abs())
    want_x = norm64(want, rms)
    # Into tensors of their own, then in place over the branch and the residual: the copies that run ahead read the
    # ends of rows that other blocks write at the same time.
    r, y = residual_norm(x, residual, post=layer, branch_scale=0.5, next_norm=rms)
    assert_rows_close(r, want, scale)
    assert_rows_close(y, want_x, 4 * want_x.abs() + 4)
    r8, (q, s) = residual_norm(x, residual, post=layer, branch_scale=0.5, next_norm=rms, quantize=True)
    assert torch.equal(r8, r) and close_int8(q, s, want_x, 1024 + 127 * 4)
    over_r, over_y = residual_norm(x, residual, post=layer, branch_scale=0.5, next_norm=rms, residual_out=residual,
                                   out=x)
    assert over_r is residual and over_y is x
    assert torch.equal(over_r, r) and torch.equal(over_y, y)
    again = rms(x)
    assert torch.equal(rms(x, out=x), again)


@pytest.mark.parametrize("rows,hidden", [(700, 2049), (1, 5120), (900, 5120), (7, 1111), (3, 100)])
@pytest.mark.parametrize("offset,pad", [(3, 5), (0, 3), (1, 0), (0, 0), (8, 8)])
def test_join_in_place_over_views(rows, hidden, offset, pad):
    """The join over its own branch and residual, as views into wider buffers: both outputs, and nothing around them."""
    size = offset + rows * (hidden + pad) + 16
    buffers = [make((size,), BF16, 20 + i) for i in range(2)]
    branch, residual = (b.as_strided((rows, hidden), (hidden + pad, 1), offset) for b in buffers)
    norm = BlockNorm(make(hidden, BF16, 3, 0.2, 1.0), make(hidden, BF16, 4, 0.2), kind="layer")
    gate = make((rows, hidden), BF16, 5)
    b = norm64(branch.double(), norm) * gate.double()
    want = residual.double() + b
    scale = torch.maximum(b.abs(), residual.double().abs())
    want_x = norm64(want, norm)
    kept = [buffer.clone() for buffer in buffers]
    r, x = residual_norm(branch, residual, post=norm, gate=gate, next_norm=norm, residual_out=residual, out=branch)
    assert r is residual and x is branch
    assert_rows_close(r, want, scale)
    assert_rows_close(x, want_x, 4 * want_x.abs() + norm.bias.double().abs() + 4)
    for now, before in zip(buffers, kept):
        now.as_strided((rows, hidden), (hidden + pad, 1), offset).zero_()
        before.as_strided((rows, hidden), (hidden + pad, 1), offset).zero_()
        assert torch.equal(now, before)


@pytest.mark.parametrize("low", [BF16, FP16])
@pytest.mark.parametrize("rows,hidden", [(3, 64), (5, 1111), (40, 5120), (2, 20000), (1, 32768)])
def test_join_of_mixed_types(rows, hidden, low):
    """An fp32 branch with parameters, gate and output of 16 bits, and a 16-bit branch with those of the other type."""
    other = FP16 if low is BF16 else BF16
    for dtype, kind in ((FP32, low), (low, other)):
        branch, residual = make((rows, hidden), dtype, 1), make((rows, hidden), FP32, 2, 3.0)
        post = BlockNorm(make(hidden, kind, 3, 0.2, 1.0))
        following = BlockNorm(make(hidden, kind, 4, 0.2, 1.0), make(hidden, kind, 5, 0.2), kind="layer")
        gate = make((rows, hidden), kind, 6)
        r, x = residual_norm(branch, residual, post=post, gate=gate, next_norm=following, out_dtype=kind)
        b = norm64(branch.double(), post) * gate.double()
        want = residual.double() + b
        assert r.dtype == FP32 and x.dtype == kind
        assert_rows_close(r, want, 3 * torch.maximum(b.abs(), residual.double().abs()))
        want_x = norm64(want, following)
        assert_rows_close(x, want_x, 4 * want_x.abs() + following.bias.double().abs() + 4)


@pytest.mark.parametrize("hidden", [64, 1111, 5120])
def test_overlaps_are_refused_unless_an_output_is_an_input(hidden):
    rows = 40
    norm = BlockNorm(make(hidden, BF16, 3, 0.2, 1.0))
    flat = make((rows * 2 * hidden + hidden,), BF16, 1)
    x = flat[:rows * hidden].view(rows, hidden)
    behind = flat[hidden:hidden + rows * hidden].view(rows, hidden)  # x, a row later
    residual = make((rows, hidden), BF16, 2)
    other = torch.empty_like(x)
    # Views side by side in wider rows are apart.
    wide = make((rows, 2 * hidden), BF16, 4)
    left, right = wide[:, :hidden], wide[:, hidden:]
    want = norm(left)
    norm(left, out=right)
    assert torch.equal(right, want)
    r, y = residual_norm(left, residual, next_norm=norm, residual_out=right, out=left)
    assert r is right and y is left
    # An output in an input's place, whichever it is.
    want = residual_norm(x, residual, next_norm=norm)
    for r_out, x_out in ((1, 0), (0, 1), (None, 1), (0, None), (1, None), (None, 0)):
        pair = [x.clone(), residual.clone()]
        got = residual_norm(*pair, next_norm=norm, residual_out=None if r_out is None else pair[r_out],
                            out=None if x_out is None else pair[x_out])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for call in (lambda: norm(x, out=behind), lambda: norm(behind, out=x),
                 lambda: norm(wide[:, 1:hidden + 1], out=left),
                 lambda: residual_norm(x, residual, residual_out=behind),
                 lambda: residual_norm(residual, x, next_norm=norm, out=behind),
                 lambda: residual_norm(x, residual, next_norm=norm, residual_out=other, out=other),
                 lambda: residual_norm(x, residual, next_norm=norm, residual_out=x, out=x),
                 lambda: residual_norm(x, residual, gate=other, residual_out=other),
                 lambda: residual_norm(x, residual, gate=other[1], next_norm=norm, out=other)):
        with pytest.raises(ValueError, match="overlaps"):
            call()


def test_outputs_that_require_a_gradient_are_refused():
    """Autograd would not see the write into a leaf (or into a tensor that a backward pass has kept)."""
    x, norm = make((4, 64), FP32, 1), BlockNorm()
    leaf = torch.zeros_like(x).requires_grad_()
    xq, xs = quantize_rows(x)
    square = torch.zeros((4, 4), device="cuda", requires_grad=True)
    for call in (lambda: norm(x, out=leaf), lambda: residual_norm(x, x, residual_out=leaf),
                 lambda: residual_norm(x, x, next_norm=norm, out=leaf), lambda: int8_linear(xq, xs, xq, xs, out=square),
                 lambda: int8_gated_linear(xq, xs, xq, xs, out=square[:, :2])):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad():
            call()
    assert torch.equal(leaf.detach(), norm(x)) or torch.equal(leaf.detach(), norm(2 * x))


def test_rows_beyond_2_to_the_31_elements():
    """Offsets of the last rows pass 32 bits: they come out as they do alone."""
    rows, hidden = 430_000, 5120
    x = torch.empty((rows, hidden), dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    norm = BlockNorm(make(hidden, BF16, 3, 0.2, 1.0))
    last = slice(rows - 70, rows)
    part = x[last].clone()
    assert torch.equal(norm(x)[last], norm(part))
    q, s = norm(x, quantize=True)
    want = norm(part, quantize=True)
    assert torch.equal(q[last], want[0]) and torch.equal(s[last], want[1])
    q, s = quantize_rows(x)
    want = quantize_rows(part)
    assert torch.equal(q[last], want[0]) and torch.equal(s[last], want[1])
    r, y = residual_norm(x, x, post=norm, next_norm=norm, residual_out=x)
    want = residual_norm(part, part, post=norm, next_norm=norm)
    assert r is x and torch.equal(r[last], want[0]) and torch.equal(y[last], want[1])


@pytest.fixture
def no_waiting():
    """Launches made inside give up at once unless their copies are there already."""
    lib = _lib.library()
    assert lib.qcc_set_wait_limit(0) == _lib.OK
    yield
    lib.qcc_set_wait_limit(2_000_000_000)
    torch.cuda.synchronize()


def given_up_or(got, want):
    """Every row is the right one or NaN all over; returns how many are NaN."""
    nan = got.isnan()
    lost = nan.all(-1)
    assert torch.equal(nan.any(-1), lost)
    assert torch.equal(got[~lost], want[~lost])
    return int(lost.sum())


@pytest.mark.parametrize("rows,hidden", [(300, 5120), (2300, 5120), (2300, 4001), (3, 20000), (700, 9000)])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_a_wait_that_runs_out_leaves_whole_rows_of_nan(rows, hidden, dtype, request):
    x, residual = make((rows, hidden), dtype, 1), make((rows, hidden), dtype, 2)
    norm = BlockNorm(make(hidden, dtype, 3, 0.1, 1.0))

    def calls():
        alone = residual_norm(x, residual, branch_scale=0.5)  # no reduction between the copies and the sum's store
        r, y = residual_norm(x, residual, post=norm, next_norm=norm)
        r8, (q, s) = residual_norm(x, residual, next_norm=norm, quantize=True)
        return [alone, r, y, r8, norm(x)], [(q, s), norm(x, quantize=True), quantize_rows(x)]

    want = calls()
    for flat in want[0]:
        assert not bool(flat.isnan().any())
    request.getfixturevalue("no_waiting")
    floats, ints = calls()
    torch.cuda.synchronize()
    for got, right in zip(floats, want[0]):
        assert given_up_or(got, right) > 0
    for (q, s), (right_q, right_s) in zip(ints, want[1]):
        lost = s.isnan()
        assert bool(lost.any()) and bool((q[lost] == 0).all())
        assert torch.equal(q[~lost], right_q[~lost]) and torch.equal(s[~lost], right_s[~lost])
    # In place, then with the ordinary bound again: nothing of the launches that gave up arrives later.
    alone = residual_norm(x, residual.clone(), branch_scale=0.5, residual_out=residual.clone())
    assert given_up_or(alone, want[0][0]) > 0
    _lib.library().qcc_set_wait_limit(2_000_000_000)
    again = calls()
    for got, right in zip(again[0], want[0]):
        assert torch.equal(got, right)
    for (q, s), (right_q, right_s) in zip(again[1], want[1]):
        assert torch.equal(q, right_q) and torch.equal(s, right_s)
