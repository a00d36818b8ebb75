"""Norms before and after an FFN block, fused with the block's gate and residual scale.

The FFN engines of this package take the normed input of their block and
return what the residual stream adds; the reference leaves the rest of the
block to the host framework (``end_to_end/model_patcher.py:12-33`` replaces
only the MLP modules).  Here that rest is one launch on each side of the FFN:

* :class:`BlockNorm` -- RMS norm or layer norm of rows, in a float type or as
  int8 rows with one scale each (the input of ``runtime.int8_dense``);
* :func:`residual_norm` -- after the block: the branch's own norm, a gate, the
  residual scales, the sum, and the next block's norm, in one pass.

All arithmetic is fp32, each output is rounded once.  Forward only.
"""
from __future__ import annotations

import torch

from .. import _lib

KINDS = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}
GATES = {None: _lib.GATE_NONE, "sigmoid": _lib.GATE_SIGMOID, "tanh": _lib.GATE_TANH}
MAX_HIDDEN = 32768


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """x [..., hidden] as rows [T, hidden], contiguous along hidden."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what} must be [..., hidden] with hidden >= 1, got {tuple(x.shape)}")
    if x.shape[-1] > MAX_HIDDEN:
        raise ValueError(f"{what} has {x.shape[-1]} values a row: at most {MAX_HIDDEN}")
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 and x.shape[1] != 1 or x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x


def _row_stride(x: torch.Tensor) -> int:
    """The row stride the C entry points take (a single row's own stride says nothing)."""
    return x.stride(0) if x.shape[0] > 1 else max(x.stride(0), x.shape[1])


def _out_rows(out: torch.Tensor | None, shape: torch.Size, rows: int, dtype: torch.dtype, device: torch.device,
              what: str) -> tuple[torch.Tensor, torch.Tensor]:
    """(the tensor to return, its rows [T, hidden])."""
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=device)
        return out, out.view(rows, shape[-1])
    if out.shape != shape or out.dtype != dtype or out.device != device:
        raise ValueError(f"{what} must be {tuple(shape)} in {dtype} on {device}")
    try:
        view = out.view(rows, shape[-1])
    except RuntimeError:
        view = None
    if view is None or (view.stride(1) != 1 and shape[-1] != 1) or (rows > 1 and view.stride(0) < shape[-1]):
        raise ValueError(f"{what} must be row-contiguous with rows one stride apart")
    return out, view


def int8_rows(rows: int, cols: int, device: torch.device) -> torch.Tensor:
    """Uninitialised int8 [rows, cols] whose rows start 16 bytes apart or a multiple of it."""
    return torch.empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=device)[:, :cols]


class BlockNorm:
    """``BlockNorm(weight, bias=None, kind="rms", eps=1e-6, weight_offset=0.0)(x)``.

    kind "rms":   x * rsqrt(mean(x^2) + eps) * (weight_offset + weight) + bias
    kind "layer": (x - mean(x)) * rsqrt(var(x) + eps) * (weight_offset + weight) + bias
    weight and bias are [hidden], contiguous, bf16 / fp16 / fp32 (one type for
    both); ``weight=None`` is a norm without a weight.  ``weight_offset=1`` is
    for models that store the weight's difference from one.
    """

    __slots__ = ("weight", "bias", "kind", "eps", "weight_offset", "hidden", "_kind", "_code", "_weight_ptr",
                 "_bias_ptr", "device")

    def __init__(self, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *, kind: str = "rms",
                 eps: float = 1e-6, weight_offset: float = 0.0):
        if kind not in KINDS:
            raise ValueError(f"kind must be one of {tuple(KINDS)}")
        if not 0 <= eps < float("inf"):
            raise ValueError("eps must be finite and not negative")
        if weight is None and weight_offset != 0.0:
            raise ValueError("weight_offset needs a weight")
        params = [p for p in (weight, bias) if p is not None]
        self.hidden, self.device, self._code = None, None, _lib.DTYPE_F32
        if params:
            self.device = _lib.require_cuda(*params)
            if any(p.dim() != 1 or not p.is_contiguous() or p.shape != params[0].shape for p in params):
                raise ValueError("weight and bias must be contiguous one-dimensional tensors of one length")
            if any(p.dtype != params[0].dtype for p in params):
                raise TypeError("weight and bias must share a dtype")
            self._code = _lib.dtype_code(params[0].dtype)
            self.hidden = params[0].shape[0]
        self.weight, self.bias, self.kind, self.eps = weight, bias, kind, float(eps)
        self.weight_offset = float(weight_offset)
        self._kind = KINDS[kind]

    def args(self, x: torch.Tensor) -> tuple:
        """The norm's C arguments for rows x, after its checks against them."""
        if self.hidden is not None:
            if self.hidden != x.shape[-1]:
                raise ValueError(f"the norm has {self.hidden} weights, its input {x.shape[-1]} values a row")
            if self.device != x.device:
                raise RuntimeError("all tensors must share a device")
        _lib.refuse_grad("BlockNorm", self.weight, self.bias)
        return (self._kind, _lib.ptr(self.weight), _lib.ptr(self.bias), self._code, self.weight_offset, self.eps)

    def __call__(self, x: torch.Tensor, *, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                 quantize: bool = False):
        """The normed rows of x [..., hidden]: a tensor like x (in out_dtype when given), or with
        ``quantize=True`` a pair (int8 [T, hidden] with rows padded to 16 bytes, fp32 scales [T]).
        ``out`` may be x itself."""
        args = self.args(x)
        return _run_norm(x, args, out, out_dtype, quantize)


_NO_NORM = (_lib.NORM_NONE, None, None, _lib.DTYPE_F32, 0.0, 0.0)


def _run_norm(x, args, out, out_dtype, quantize):
    device = _lib.require_cuda(x)
    code = _lib.dtype_code(x.dtype)
    _lib.refuse_grad("BlockNorm", x)
    rows = _rows(x, "x")
    t, hidden = rows.shape
    scale = None
    if quantize:
        if out is not None or out_dtype is not None:
            raise ValueError("quantize=True returns its own int8 rows: out and out_dtype do not apply")
        out = out_rows = int8_rows(t, hidden, device)
        scale = torch.empty(t, dtype=torch.float32, device=device)
        out_code = _lib.DTYPE_I8
    else:
        dtype = out_dtype or (x.dtype if out is None else out.dtype)
        out_code = _lib.dtype_code(dtype)
        out, out_rows = _out_rows(out, x.shape, t, dtype, device, "out")
    lib = _lib.library()
    status = _lib.on_device(device, lib.qcc_norm_rows, rows.data_ptr(), _row_stride(rows), code, t, hidden, *args,
                            out_rows.data_ptr(), _row_stride(out_rows), out_code, _lib.ptr(scale),
                            _lib.stream_handle(device))
    if status:
        _lib.check(status, "qcc_norm_rows")
    return (out, scale) if quantize else out


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., cols] in bf16 / fp16 / fp32 -> (int8 [T, cols], fp32 scales [T]), one symmetric scale a row.

    scale = amax / 127 and q = round_half_even(x * (127 / amax)).  A row with
    amax < 2^-119 gets scale 0 and zeros; one that holds a NaN or an infinity
    gets scale NaN and zeros, so every product with it is NaN.  The int8 rows
    are padded to a multiple of 16 bytes, as ``runtime.int8_dense`` wants them.
    """
    return _run_norm(x, _NO_NORM, None, None, True)


def _gate_args(gate: torch.Tensor | None, activation: str | None, shape: torch.Size) -> tuple:
    """(gate kept alive, C arguments): the gate as rows of 1 or hidden values, each used by consecutive rows of x."""
    if activation not in GATES:
        raise ValueError(f"gate_activation must be one of {tuple(GATES)}")
    if gate is None:
        return None, (None, 0, 1, 1, _lib.DTYPE_F32, _lib.GATE_NONE)
    code = _lib.dtype_code(gate.dtype)
    cols = gate.shape[-1] if gate.dim() else 1
    lead = list(gate.shape[:-1])
    x_lead = list(shape[:-1])
    if cols not in (1, shape[-1]) or len(lead) > len(x_lead):
        raise ValueError(f"gate {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
    # Rows shared by the trailing leading axes (per sequence, or one row for all), full before them.
    lead = [1] * (len(x_lead) - len(lead)) + lead
    each = 1
    while lead and (lead[-1] == 1):
        lead.pop()
        each *= x_lead[len(lead)]
    if lead != x_lead[:len(lead)]:
        raise ValueError(f"gate {tuple(gate.shape)} does not broadcast to {tuple(shape)} along its last axes")
    rows = gate.reshape(-1, cols)
    if rows.stride(1) != 1 or rows.stride(0) < cols:
        rows = rows.contiguous()
    return rows, (rows.data_ptr(), rows.stride(0), max(each, 1), cols, code, GATES[activation])


def residual_norm(branch: torch.Tensor, residual: torch.Tensor, *, post: BlockNorm | None = None,
                  gate: torch.Tensor | None = None, gate_activation: str | None = None, residual_scale: float = 1.0,
                  branch_scale: float = 1.0, next_norm: BlockNorm | None = None, quantize: bool = False,
                  residual_out: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  out_dtype: torch.dtype | None = None):
    """The end of one block and the start of the next, in one launch.

    r = residual_scale * residual + branch_scale * act(gate) * post(branch)
    x = next_norm(r)

    branch, residual [..., hidden]; residual in branch's dtype or fp32, and r
    comes back in it.  gate: a tensor whose last axis is 1 or hidden and whose
    leading axes match branch's, with trailing ones of them allowed to be 1 or
    missing altogether ([hidden], [T, 1], [T, hidden], [B, 1, hidden], ...).
    Returns r without a ``next_norm``, else (r, x), or (r, (int8, scales)) with
    ``quantize=True``.  ``residual_out`` may be residual (in place) and ``out``
    branch; other overlaps of inputs and outputs are not supported.
    """
    device = _lib.require_cuda(branch, residual, gate)
    if residual.shape != branch.shape:
        raise ValueError(f"residual {tuple(residual.shape)} must have branch's shape {tuple(branch.shape)}")
    code = _lib.dtype_code(branch.dtype)
    if residual.dtype != branch.dtype and residual.dtype != torch.float32:
        raise TypeError("residual must be in branch's dtype or float32")
    _lib.refuse_grad("residual_norm", branch, residual, gate)
    if next_norm is None and (quantize or out is not None or out_dtype is not None):
        raise ValueError("quantize, out and out_dtype need a next_norm")
    shape = branch.shape
    post_args = _NO_NORM if post is None else post.args(branch)
    next_args = _NO_NORM if next_norm is None else next_norm.args(branch)
    gate_rows, gate_args = _gate_args(gate, gate_activation, shape)
    rows, res_rows = _rows(branch, "branch"), _rows(residual, "residual")
    t, hidden = rows.shape
    residual_out, res_out_rows = _out_rows(residual_out, shape, t, residual.dtype, device, "residual_out")
    scale, out_ptr, ld_out, out_code = None, None, hidden, code
    if next_norm is not None:
        if quantize:
            if out is not None or out_dtype is not None:
                raise ValueError("quantize=True returns its own int8 rows: out and out_dtype do not apply")
            out = out_rows = int8_rows(t, hidden, device)
            scale = torch.empty(t, dtype=torch.float32, device=device)
            out_code = _lib.DTYPE_I8
        else:
            dtype = out_dtype or (branch.dtype if out is None else out.dtype)
            out_code = _lib.dtype_code(dtype)
            out, out_rows = _out_rows(out, shape, t, dtype, device, "out")
        out_ptr, ld_out = out_rows.data_ptr(), _row_stride(out_rows)
    lib = _lib.library()
    status = _lib.on_device(device, lib.qcc_residual_norm, rows.data_ptr(), _row_stride(rows), code,
                            res_rows.data_ptr(), _row_stride(res_rows), _lib.dtype_code(residual.dtype), t, hidden,
                            *post_args, *gate_args, float(residual_scale), float(branch_scale),
                            res_out_rows.data_ptr(), _row_stride(res_out_rows), *next_args, out_ptr, ld_out, out_code,
                            _lib.ptr(scale), _lib.stream_handle(device))
    if status:
        _lib.check(status, "qcc_residual_norm")
    if next_norm is None:
        return residual_out
    return residual_out, ((out, scale) if quantize else out)
