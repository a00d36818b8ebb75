"""The dense FFN in 8-bit integers: one scale per token and one per output channel.

The reference's dense form of a layer (``runtime/ffn.py:11-17``, the form its
bridge falls back to for prompts and for layers without a selector) runs three
projections in the model's float type.  Here the weights are int8 rows with an
fp32 scale a channel (half of bf16's bytes) and the activations int8 rows with
a scale a token; the integer sums are exact, the scales, the bias and silu are
applied in fp32 on the accumulators, and the output is rounded once.

* :func:`quantize_rows` -- rows to int8, for activations and (once) weights;
  ``BlockNorm(...)(x, quantize=True)`` writes the same form from the norm;
* :func:`int8_linear` and :func:`int8_gated_linear` -- the products, on int8;
* :class:`Int8Linear`, :class:`Int8GatedLinear` -- a weight with its scales;
* :class:`Int8GatedFFN` -- the whole layer.

Forward only.
"""
from __future__ import annotations

import torch

from .. import _lib
from .block_norm import int8_rows, quantize_rows
from .packing import PackedFFNWeights, validate_weight_shapes

_raw_stream, _current_device, _forward_ad = _lib.raw_stream, _lib.current_device, _lib.forward_ad
MAX_COLS = 131071       # |q| <= 128: the int32 sums cannot overflow
MAX_TOKENS = 1 << 20
MAX_CHANNELS = 1 << 19


_INT8, _FLOAT32 = torch.int8, torch.float32


def _int8_operand(q: torch.Tensor, scale: torch.Tensor, what: str) -> tuple[int, int, int]:
    """Checks an int8 matrix with its row scales; returns its rows, columns and row stride."""
    if q.dim() != 2 or q.dtype is not _INT8:
        raise ValueError(f"{what} must be an int8 matrix")
    rows, cols = q.shape
    ld, step = q.stride()
    if step != 1 and cols != 1:
        raise ValueError(f"{what} must be contiguous along its columns")
    if scale.dtype is not _FLOAT32 or scale.shape != (rows,) or not scale.is_contiguous():
        raise ValueError(f"the scales of {what} must be a contiguous float32 tensor with one value per row")
    if rows <= 1:
        ld = cols + -cols % 16
    if ld & 15 or q.data_ptr() & 15 or ld < cols:
        raise ValueError(f"the rows of {what} must start on multiples of 16 bytes (quantize_rows stores them so)")
    return rows, cols, ld


def _products(xq, x_scale, wq, w_scale, bias, out, out_dtype, gated):
    tokens, cols, ldx = _int8_operand(xq, x_scale, "x")
    rows, w_cols, ldw = _int8_operand(wq, w_scale, "w")
    index = xq.get_device()
    if (index < 0 or x_scale.get_device() != index or wq.get_device() != index or w_scale.get_device() != index
            or (bias is not None and bias.get_device() != index) or (out is not None and out.get_device() != index)):
        _lib.require_cuda(xq, x_scale, wq, w_scale, bias, out)
    if w_cols != cols:
        raise ValueError(f"x has {cols} columns, w {w_cols}")
    if gated and rows & 1:
        raise ValueError("a gated weight has as many up rows as gate rows")
    channels = rows >> 1 if gated else rows
    if channels < 1 or cols < 1:
        raise ValueError("w must have rows and columns")
    if cols > MAX_COLS or tokens > MAX_TOKENS or channels > MAX_CHANNELS:
        raise ValueError(f"at most {MAX_TOKENS} tokens, {MAX_CHANNELS} channels and {MAX_COLS} columns")
    if (x_scale.requires_grad or w_scale.requires_grad or (bias is not None and bias.requires_grad)
            or _forward_ad._current_level >= 0):
        _lib.refuse_grad("the int8 product", x_scale, w_scale, bias)
    if out is None:
        if out_dtype is None:
            out_dtype = torch.bfloat16
        y_code = _lib.dtype_code(out_dtype)
        out = torch.empty(tokens, channels, dtype=out_dtype, device=xq.device)
        ldy = channels
    else:
        y_code = _lib.dtype_code(out.dtype)
        if out.requires_grad:
            _lib.refuse_grad("writing out", out)
        if (out.shape != (tokens, channels) or (out_dtype or out.dtype) != out.dtype
                or (out.stride(1) != 1 and channels != 1) or (tokens > 1 and out.stride(0) < channels)):
            raise ValueError("out must be a row-contiguous [tokens, channels] tensor of out_dtype")
        ldy = max(out.stride(0), channels)
    lib = _lib.library()
    if gated:
        args = (xq.data_ptr(), ldx, x_scale.data_ptr(), wq.data_ptr(), ldw, w_scale.data_ptr(), tokens, channels, cols,
                out.data_ptr(), ldy, y_code)
        fn = lib.qcc_int8_gated_linear
    else:
        bias_ptr, bias_code = None, _lib.DTYPE_F32
        if bias is not None:
            if bias.dim() != 1 or bias.shape[0] != channels or not bias.is_contiguous():
                raise ValueError("bias must be a contiguous tensor with one value per channel")
            bias_ptr, bias_code = bias.data_ptr(), _lib.dtype_code(bias.dtype)
        args = (xq.data_ptr(), ldx, x_scale.data_ptr(), wq.data_ptr(), ldw, w_scale.data_ptr(), bias_ptr, bias_code,
                tokens, channels, cols, out.data_ptr(), ldy, y_code)
        fn = lib.qcc_int8_linear
    status = fn(*args, _raw_stream(index)) if _current_device() == index else _lib.launch(index, fn, *args)
    if status:
        _lib.check(status, "qcc_int8_gated_linear" if gated else "qcc_int8_linear")
    return out


def int8_linear(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, *,
                bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """y [T, N] = (xq @ wq.T) * x_scale[:, None] * w_scale + bias, in out_dtype (bf16 by default).

    xq int8 [T, K] and wq int8 [N, K] with rows on multiples of 16 bytes, their
    scales fp32 [T] and [N]; bias [N] in bf16, fp16 or fp32.
    """
    return _products(xq, x_scale, wq, w_scale, bias, out, out_dtype, False)


def int8_gated_linear(xq: torch.Tensor, x_scale: torch.Tensor, wq: torch.Tensor, w_scale: torch.Tensor, *,
                      out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """h [T, N] = silu(g) * u with g, u the products of xq with the first and the last N rows of wq [2N, K]."""
    return _products(xq, x_scale, wq, w_scale, None, out, out_dtype, True)


def _rows_of(x, cols: int) -> tuple[torch.Tensor, torch.Tensor, torch.Size]:
    """(int8 rows, scales, leading shape) of a float tensor [..., cols] or of a pair already quantised."""
    if isinstance(x, tuple):
        q, scale = x
        lead = q.shape[:-1]
    else:
        lead = x.shape[:-1]
        if x.dim() < 1 or x.shape[-1] != cols:
            raise ValueError(f"x must be [..., {cols}], got {tuple(x.shape)}")
        q, scale = quantize_rows(x)
    return q, scale, lead


class Int8Linear:
    """``Int8Linear(wq, w_scale, bias=None)(x)``: a projection whose weight [N, K] is int8 rows with scales.

    x is a float tensor [..., K], quantised per row on the way, or a pair
    (int8 [T, K], scales [T]); the result is [..., N] in ``out_dtype`` (the
    dtype of a float x, else bf16).
    """

    gated = False

    def __init__(self, weight: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None):
        _int8_operand(weight, scale, "w")
        _lib.require_cuda(weight, scale, bias)
        self.weight, self.scale, self.bias = weight, scale, bias
        self.rows, self.cols = weight.shape

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: torch.Tensor | None = None) -> "Int8Linear":
        """From a float weight [N, K], quantised per output channel."""
        if weight.dim() != 2:
            raise ValueError("weight must be a matrix")
        return cls(*quantize_rows(weight.detach()), bias)

    def __call__(self, x, *, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        q, scale, lead = _rows_of(x, self.cols)
        if out_dtype is None and not isinstance(x, tuple):
            out_dtype = x.dtype
        y = _products(q, scale, self.weight, self.scale, self.bias, None, out_dtype, self.gated)
        return y if len(lead) == 1 else y.view(*lead, y.shape[1])


class Int8GatedLinear(Int8Linear):
    """``silu(x @ gate.T) * (x @ up.T)`` with one int8 weight [2N, K]: the gate rows, then the up rows."""

    gated = True

    def __init__(self, weight: torch.Tensor, scale: torch.Tensor):
        super().__init__(weight, scale)
        if self.rows % 2:
            raise ValueError("a gated weight has as many up rows as gate rows")

    @classmethod
    def from_weights(cls, gate: torch.Tensor, up: torch.Tensor) -> "Int8GatedLinear":
        """From float gate and up projections [N, K], quantised per row."""
        if gate.dim() != 2 or gate.shape != up.shape or gate.dtype != up.dtype:
            raise ValueError("gate and up must be matrices of one shape and dtype")
        n, k = gate.shape
        weight = int8_rows(2 * n, k, gate.device)
        scale = torch.empty(2 * n, dtype=torch.float32, device=gate.device)
        for begin, part in ((0, gate), (n, up)):
            q, s = quantize_rows(part.detach())
            weight[begin:begin + n] = q
            scale[begin:begin + n] = s
        return cls(weight, scale)

    @classmethod
    def from_packed(cls, weights: PackedFFNWeights) -> "Int8GatedLinear":
        """From the gate and up parts of packed records (``OracleModeFFN(..., gate_up=...)`` takes the result)."""
        h, hp = weights.hidden, weights.hidden_pad
        return cls.from_weights(weights.packed[:, :h], weights.packed[:, hp:hp + h])

    @classmethod
    def from_weight(cls, weight: torch.Tensor, bias: torch.Tensor | None = None) -> "Int8GatedLinear":
        """From a float weight [2N, K]: the gate rows, then the up rows."""
        if bias is not None:
            raise ValueError("a gated projection has no bias")
        if weight.dim() != 2:
            raise ValueError("weight must be a matrix")
        return cls(*quantize_rows(weight.detach()))


class Int8GatedFFN:
    """The dense gated FFN of one layer: y = down(silu(gate x) * up x), every projection in int8.

    The dense counterpart of ``IndexedSparseFFN`` (reference runtime/ffn.py:11-17):
    quantise rows, gate | up product, quantise rows, down product.  The gated
    activation is stored in bf16 between the two (fp32 for fp32 outputs): its
    rounding, 2^-9, is below half a quantisation step of the row's largest
    values, and fp16's range could overflow.
    """

    def __init__(self, gate_up: Int8GatedLinear, down: Int8Linear):
        if down.cols != gate_up.rows // 2 or down.gated:
            raise ValueError(f"down takes {down.cols} values, gate and up give {gate_up.rows // 2}")
        self.gate_up, self.down = gate_up, down

    @classmethod
    def from_weights(cls, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor,
                     transposed_down: bool = False) -> "Int8GatedFFN":
        """From gate, up [N, H] and down [H, N] (or its transpose), as ``pack_neuron_major`` takes them."""
        validate_weight_shapes(gate, up, down, transposed_down)
        return cls(Int8GatedLinear.from_weights(gate, up),
                   Int8Linear.from_weight(down.t() if transposed_down else down))

    @property
    def hidden(self) -> int:
        return self.gate_up.cols

    @property
    def intermediate(self) -> int:
        return self.down.cols

    def __call__(self, x, *, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """y [..., H] for a float x [..., H] or a pair (int8 rows, scales)."""
        if out_dtype is None:
            out_dtype = torch.bfloat16 if isinstance(x, tuple) else x.dtype
        between = torch.float32 if out_dtype == torch.float32 else torch.bfloat16
        return self.down(self.gate_up(x, out_dtype=between), out_dtype=out_dtype)
