"""The layer's FFN half (FFNBlock) and the oracle mode's int8 gate | up pass, against their parts and float64."""
from __future__ import annotations

import pytest
import torch

import conftest  # noqa: F401
from qcc_b200.runtime import (BlockNorm, FFNBlock, IndexedSparseFFN, Int8GatedFFN, Int8GatedLinear, quantize_rows,
                              residual_norm, select_topk)
from qcc_b200.runtime.oracle_mode import OracleModeFFN
from qcc_b200.runtime.packing import pack_neuron_major

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def layer(hidden, inner, dtype, seed):
    gen = torch.Generator().manual_seed(seed)

    def make(*shape, scale):
        return (torch.randn(shape, generator=gen) * scale).to(dtype).cuda()

    return make(inner, hidden, scale=0.06), make(inner, hidden, scale=0.06), make(hidden, inner, scale=0.04), gen


def norm(hidden, dtype, gen):
    return BlockNorm((1 + 0.1 * torch.randn(hidden, generator=gen)).to(dtype).cuda())


@pytest.mark.parametrize("tokens", [1, 3])
@pytest.mark.parametrize("res_dtype", [torch.bfloat16, torch.float32])
def test_block_around_the_indexed_ffn(tokens, res_dtype):
    hidden, inner = 264, 512
    gate, up, down, gen = layer(hidden, inner, torch.bfloat16, 0)
    engine = IndexedSparseFFN(pack_neuron_major(gate, up, down))
    ids = torch.randperm(inner, generator=gen)[:200].sort().values.to(torch.int32).cuda()
    pre, post, following = (norm(hidden, torch.bfloat16, gen) for _ in range(3))
    residual = torch.randn(tokens, hidden, generator=gen).to(res_dtype).cuda()
    token_gate = torch.randn(tokens, 1, generator=gen).bfloat16().cuda()
    block = FFNBlock(engine, pre, post, next_norm=following, gate_activation="sigmoid", branch_scale=0.5,
                     dtype=torch.bfloat16)
    r, x = block(residual, ids, gate=token_gate)
    assert r.dtype == res_dtype and x.dtype == torch.bfloat16
    y = engine(pre(residual, out_dtype=torch.bfloat16), ids)
    want = residual_norm(y, residual, post=post, gate=token_gate, gate_activation="sigmoid", branch_scale=0.5,
                         next_norm=following)
    assert torch.equal(r, want[0]) and torch.equal(x, want[1])
    # The next block may take x instead of norming the residual again.
    second = FFNBlock(engine, following)
    assert torch.equal(second(r, ids, x=x), residual_norm(engine(x, ids), r))
    # float64 of the join, from the FFN's own output.
    branch = y.double() / (y.double().square().mean(-1, keepdim=True) + post.eps).sqrt() * post.weight.double()
    exact = residual.double() + 0.5 * token_gate.double().sigmoid() * branch
    half = torch.finfo(res_dtype).eps / 2
    scale = exact.abs().amax(1, keepdim=True) + branch.abs().amax(1, keepdim=True)
    assert bool(((r.double() - exact).abs() <= half * exact.abs() + 256 * U32 * scale).all())


@pytest.mark.parametrize("tokens", [1, 70])
def test_block_around_the_int8_ffn(tokens):
    hidden, inner = 264, 520
    gate, up, down, gen = layer(hidden, inner, torch.bfloat16, 1)
    ffn = Int8GatedFFN.from_weights(gate, up, down)
    pre, following = norm(hidden, torch.bfloat16, gen), norm(hidden, torch.bfloat16, gen)
    residual = torch.randn(tokens, hidden, generator=gen).bfloat16().cuda()
    block = FFNBlock(ffn, pre, next_norm=following, quantize_next=True)
    r, (q, s) = block(residual)
    y = ffn(pre(residual, quantize=True))
    want, (wq, ws) = residual_norm(y, residual, next_norm=following, quantize=True)
    assert torch.equal(r, want) and torch.equal(q, wq) and torch.equal(s, ws)
    again = FFNBlock(ffn, following)(r, x=(q, s))
    assert torch.equal(again, residual_norm(ffn((q, s)), r))
    with pytest.raises(ValueError, match="next_norm"):
        FFNBlock(ffn, pre, quantize_next=True)


@pytest.mark.parametrize("tokens,hidden,inner,dtype", [(1, 256, 512, torch.bfloat16), (11, 200, 300, torch.float16),
                                                       (130, 256, 700, torch.float32)])
def test_oracle_mode_with_int8_gate_up(tokens, hidden, inner, dtype):
    gate, up, down, gen = layer(hidden, inner, dtype, 2)
    weights = pack_neuron_major(gate, up, down)
    gate_up = Int8GatedLinear.from_packed(weights)
    whole = Int8GatedLinear.from_weights(gate, up)
    assert torch.equal(gate_up.weight, whole.weight) and torch.equal(gate_up.scale, whole.scale)
    x = torch.randn(tokens, hidden, generator=gen).to(dtype).cuda()
    plain = OracleModeFFN(weights, 0.25)
    mode = OracleModeFFN(weights, 0.25, gate_up=gate_up)
    acts = mode.activations(x)
    q, s = quantize_rows(x)
    both = (q.double() @ gate_up.weight.double().t()) * s.double()[:, None] * gate_up.scale.double()
    g, u = both[:, :inner], both[:, inner:]
    want = torch.nn.functional.silu(g) * u
    # g and u carry 3 roundings each; silu and the product 10, and exp 4 |g| (see the int8 products' tests).
    assert bool(((acts.double() - want).abs() <= want.abs() * (17 + 4 * g.abs()) * U32 + 2.0 ** -119 * u.abs()).all())
    y, ids = mode(x)
    assert ids.shape == (tokens, mode.k)
    importance = acts.abs() * mode.column_weights
    assert torch.equal(ids, select_topk(importance, mode.k))
    assert torch.equal(y, mode.down(acts, ids))
    # Near the records' own oracle: int8 moves an activation by about 1 % of its row's norm.
    exact = plain.activations(x)
    assert float((acts - exact).norm() / exact.norm()) < 0.05
    with pytest.raises(ValueError, match="gate_up"):
        OracleModeFFN(weights, 0.25, gate_up=Int8GatedLinear.from_weights(gate[:inner // 2], up[:inner // 2]))
