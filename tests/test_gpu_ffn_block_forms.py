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
