"""FFNBlock around every FFN of the package, and with every shape of the residual."""
from __future__ import annotations

import pytest
import torch

import conftest  # noqa: F401
from qcc_b200.runtime import FFNBlock, Int8GatedFFN, Int8GatedLinear, IndexedSparseFFN, residual_norm
from qcc_b200.runtime.ffn import TorchDynamicSparseFFN
from qcc_b200.runtime.oracle_mode import OracleModeFFN
from qcc_b200.runtime.packing import pack_neuron_major
from qcc_b200.runtime.prefill import BlockSparsePrefill
from qcc_b200.runtime.sharded import ShardedIndexedFFN
from test_gpu_ffn_block import layer, norm

pytestmark = pytest.mark.gpu

BF16, FP32 = torch.bfloat16, torch.float32
HIDDEN, INNER = 256, 512


def assert_same(got, want):
    """Tensors, and tuples of them, equal bit for bit and in shape."""
    if isinstance(want, tuple):
        assert isinstance(got, tuple) and len(got) == len(want)
        for g, w in zip(got, want):
            assert_same(g, w)
    else:
        assert got.shape == want.shape and got.dtype == want.dtype and torch.equal(got, want)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("tokens", [1, 11])
def test_block_around_the_oracle_mode(tokens, int8):
    gate, up, down, gen = layer(HIDDEN, INNER, BF16, 0)
    weights = pack_neuron_major(gate, up, down)
    mode = OracleModeFFN(weights, 0.25, gate_up=Int8GatedLinear.from_packed(weights) if int8 else None)
    pre, post, following = (norm(HIDDEN, BF16, gen) for _ in range(3))
    residual = torch.randn(tokens, HIDDEN, generator=gen).bfloat16().cuda()
    y, ids = mode(pre(residual))
    assert ids.shape == (tokens, mode.k)
    got = FFNBlock(mode, pre, post, next_norm=following, branch_scale=0.5)(residual)
    assert_same(got, residual_norm(y, residual, post=post, next_norm=following, branch_scale=0.5))


@pytest.mark.parametrize("shape", [(3,), (2, 3), (2, 1, 2), (), (0, 4), (0,)])
@pytest.mark.parametrize("kind", ["indexed", "module", "oracle", "prefill", "sharded", "int8", "callable"])
def test_every_shape_of_the_residual(kind, shape):
    """A residual of any leading axes gives what its rows give, with int8 and float inputs of the next block."""
    gate, up, down, gen = layer(HIDDEN, INNER, BF16, 1)
    weights = pack_neuron_major(gate, up, down)
    ids = torch.randperm(INNER, generator=gen)[:128].sort().values.to(torch.int32).cuda()
    tokens = 1
    for n in shape:
        tokens *= n
    seen = []

    def plain(x):
        seen.append(x.shape)
        return x * 2

    ffn, args = {"indexed": lambda: (IndexedSparseFFN(weights), (ids,)),
                 "module": lambda: (TorchDynamicSparseFFN(gate, up, down), (ids,)),
                 "oracle": lambda: (OracleModeFFN(weights, 0.25), ()),
                 "prefill": lambda: (BlockSparsePrefill(weights), ([[0, 2]],)),
                 "sharded": lambda: (ShardedIndexedFFN(weights, allreduce="nccl"), (ids,)),
                 "int8": lambda: (Int8GatedFFN.from_weights(gate, up, down), ()),
                 "callable": lambda: (plain, ())}[kind]()
    if tokens == 0 and kind in ("prefill", "oracle", "sharded"):
        pytest.skip("these FFNs take one token at least")
    pre, post, following = (norm(HIDDEN, BF16, gen) for _ in range(3))
    residual = torch.randn(*shape, HIDDEN, generator=gen).bfloat16().cuda()
    rows = residual.reshape(-1, HIDDEN)
    token_gate = torch.randn(*shape, 1, generator=gen).bfloat16().cuda()
    for quantize in (False, True):
        block = FFNBlock(ffn, pre, post, next_norm=following, quantize_next=quantize, gate_activation="sigmoid")
        want_r, want_x = block(rows, *args, gate=token_gate.reshape(-1, 1))
        r, x = block(residual, *args, gate=token_gate)
        assert_same(r, want_r.view(residual.shape))
        assert_same(x, want_x if quantize else want_x.view(residual.shape))
    # x made by the block before: with the residual's axes, or int8 rows.
    given = pre(residual, quantize=True) if kind == "int8" else pre(residual)
    assert_same(FFNBlock(ffn, pre, post)(residual, *args, x=given),
                FFNBlock(ffn, pre, post)(rows, *args).view(residual.shape))
    if kind == "callable":
        assert residual.shape in seen
