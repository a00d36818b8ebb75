"""The FFN half of a decoder layer around any of this package's FFNs.

``FFNBlock(ffn, pre, post)(residual, ...)`` is

    x  = pre(residual)
    y  = ffn(x, ...)
    r  = residual_scale * residual + branch_scale * act(gate) * post(y)

and, with ``next_norm``, also the next block's input next_norm(r), made in the
launch that makes r.  The reference leaves this half to the model it patches
(``end_to_end/model_patcher.py:12-33``).
"""
from __future__ import annotations

import torch

from .block_norm import BlockNorm, residual_norm
from .engine import IndexedSparseFFN
from .ffn import TorchDynamicSparseFFN
from .int8_dense import Int8GatedFFN
from .oracle_mode import OracleModeFFN
from .prefill import BlockSparsePrefill
from .sharded import ShardedIndexedFFN

# FFNs that take rows [T, hidden] only; other callables get x with the residual's leading axes.
_OF_ROWS = IndexedSparseFFN, TorchDynamicSparseFFN, OracleModeFFN, BlockSparsePrefill, ShardedIndexedFFN


class FFNBlock:
    """Norm, FFN, norm, gate and residual sum of one layer.

    ffn: a callable y = ffn(x, *args, **kwargs) -- ``IndexedSparseFFN`` (args:
    the selected ids), ``BlockSparsePrefill`` (the tiles' blocks),
    ``Int8GatedFFN`` (none), ...  An ``Int8GatedFFN`` gets pre's int8 rows.  Of
    a tuple (``OracleModeFFN``: y and its ids) the first item is y.
    dtype: the type of x (and of y) when it is not the residual's, e.g. bf16
    records under an fp32 residual.  ``quantize_next``: next_norm(r) as int8
    rows, for a next block that takes them.
    """

    def __init__(self, ffn, pre: BlockNorm, post: BlockNorm | None = None, *, next_norm: BlockNorm | None = None,
                 quantize_next: bool = False, gate_activation: str | None = None, residual_scale: float = 1.0,
                 branch_scale: float = 1.0, dtype: torch.dtype | None = None):
        if quantize_next and next_norm is None:
            raise ValueError("quantize_next needs a next_norm")
        self.ffn, self.pre, self.post, self.next_norm = ffn, pre, post, next_norm
        self.quantize_next, self.gate_activation = quantize_next, gate_activation
        self.residual_scale, self.branch_scale, self.dtype = float(residual_scale), float(branch_scale), dtype

    def __call__(self, residual: torch.Tensor, *args, x=None, gate: torch.Tensor | None = None, **kwargs):
        """r, or (r, next input) with a next_norm, for residual [..., hidden] (int8 next inputs are rows [T, hidden]).

        x: pre(residual) when the previous block made it (its next_norm's
        output; int8 rows for an ``Int8GatedFFN``); args and kwargs go to ffn,
        whose tokens are the residual's rows in order.
        """
        dtype = self.dtype or residual.dtype
        int8 = isinstance(self.ffn, Int8GatedFFN)
        if x is None:
            x = self.pre(residual, quantize=True) if int8 else self.pre(residual, out_dtype=dtype)
        if int8:
            kwargs.setdefault("out_dtype", dtype)
        elif isinstance(self.ffn, _OF_ROWS) and x.dim() != 2:
            x = x.reshape(-1, x.shape[-1])
        y = self.ffn(x, *args, **kwargs)
        if isinstance(y, tuple):
            y = y[0]
        if int8 or isinstance(self.ffn, _OF_ROWS):
            y = y.reshape(residual.shape)
        return residual_norm(y, residual, post=self.post, gate=gate, gate_activation=self.gate_activation,
                             residual_scale=self.residual_scale, branch_scale=self.branch_scale,
                             next_norm=self.next_norm, quantize=self.quantize_next)
