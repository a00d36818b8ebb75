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

import ctypes

import torch

from .. import _lib

_raw_stream, _current_device, _forward_ad = _lib.raw_stream, _lib.current_device, _lib.forward_ad
KINDS = {"rms": _lib.NORM_RMS, "layer": _lib.NORM_LAYER}
GATES = {None: _lib.GATE_NONE, "sigmoid": _lib.GATE_SIGMOID, "tanh": _lib.GATE_TANH}
MAX_HIDDEN = 32768
MAX_QUANTIZED = 131071  # columns of rows that are quantised as they are: as many as the int8 products take
MAX_ROWS = 2 ** 31 - 1


def _check_hidden(x: torch.Tensor, what: str, most: int = MAX_HIDDEN) -> None:
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what} must be [..., hidden] with hidden >= 1, got {tuple(x.shape)}")
    if x.shape[-1] > most:
        raise ValueError(f"{what} has {x.shape[-1]} values a row: at most {most}")


def _rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """x [..., hidden] as rows [T, hidden] contiguous along hidden, and their stride."""
    if x.is_contiguous():
        return x, x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 or x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x, x.stride(0)


def _out_rows(out: torch.Tensor, shape: torch.Size, rows: int, dtype: torch.dtype, index: int, what: str) -> int:
    """Checks a caller's output tensor; returns the stride of its rows."""
    if out.requires_grad:
        _lib.refuse_grad(f"writing {what}", out)
    if out.shape != shape or out.dtype != dtype or out.get_device() != index:
        raise ValueError(f"{what} must be {tuple(shape)} in {dtype} on the inputs' device")
    hidden = shape[-1]
    if out.is_contiguous():
        return hidden
    try:
        view = out.view(rows, hidden)
    except RuntimeError:
        view = None
    if view is None or (view.stride(1) != 1 and hidden != 1) or (rows > 1 and view.stride(0) < hidden):
        raise ValueError(f"{what} must be row-contiguous with rows one stride apart")
    return max(view.stride(0), hidden)


def _overlap(a: tuple, b: tuple) -> bool:
    """Whether rows given as (address, bytes between rows, bytes of a row, rows) share memory.  Rows of two different
    strides, neither of them dense, may be interleaved in any way: taken as apart."""
    (pa, sa, na, ta), (pb, sb, nb, tb) = a, b
    if pb >= pa + (ta - 1) * sa + na or pa >= pb + (tb - 1) * sb + nb or not (ta and tb):
        return False
    if sa == sb and ta > 1 and tb > 1:
        apart = (pb - pa) % sa  # views side by side in wider rows
        return apart < na or apart + nb > sa
    for (p, s, n, t), (q, r, m, u) in ((a, b), (b, a)):
        if t == 1 or s == n:  # dense: the first of the other's rows that ends behind its start
            i = max(0, (p - q - m) // r + 1) if u > 1 else 0
            return i < u and q + i * r < p + (t - 1) * s + n
    return False


def _extent(x: torch.Tensor, ld: int, cols: int, rows: int) -> tuple:
    size = x.itemsize
    return x.data_ptr(), (ld if rows > 1 else cols) * size, cols * size, rows


def _check_overlap(out: tuple, name: str, inputs: tuple) -> None:
    """An output may be an input itself (its rows and type), or apart from it."""
    for what, rows in inputs:
        if rows is not None and out != rows and _overlap(out, rows):
            raise ValueError(f"{name} overlaps {what} without being it")


def int8_rows(rows: int, cols: int, device: torch.device) -> torch.Tensor:
    """Uninitialised int8 [rows, cols] whose rows start on multiples of 16 bytes."""
    pad = -cols % 16
    if pad:
        return torch.empty_strided((rows, cols), (cols + pad, 1), dtype=torch.int8, device=device)
    return torch.empty(rows, cols, dtype=torch.int8, device=device)


class BlockNorm:
    """``BlockNorm(weight, bias=None, kind="rms", eps=1e-6, weight_offset=0.0)(x)``.

    kind "rms":   x * rsqrt(mean(x^2) + eps) * (weight_offset + weight) + bias
    kind "layer": (x - mean(x)) * rsqrt(var(x) + eps) * (weight_offset + weight) + bias
    weight and bias are [hidden], contiguous, bf16 / fp16 / fp32 (one type for
    both); ``weight=None`` is a norm without a weight.  ``weight_offset=1`` is
    for models that store the weight's difference from one.
    """

    __slots__ = ("weight", "bias", "_constants", "_bound")

    def __init__(self, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *, kind: str = "rms",
                 eps: float = 1e-6, weight_offset: float = 0.0):
        if kind not in KINDS:
            raise ValueError(f"kind must be one of {tuple(KINDS)}")
        if not 0 <= eps < float("inf"):
            raise ValueError("eps must be finite and not negative")
        self.weight, self.bias = weight, bias
        self._constants = KINDS[kind], weight_offset, eps
        self._bind()

    def _bind(self) -> tuple:
        """Checks weight and bias as they are now and makes the C argument of them.  It is replaced, never rewritten:
        another thread may be launching with the one before."""
        weight, bias = self.weight, self.bias
        if weight is None and self._constants[1] != 0.0:
            raise ValueError("weight_offset needs a weight")
        hidden, index, dtype, code = None, None, None, _lib.DTYPE_F32
        for p in (weight, bias):
            if p is None:
                continue
            if p.get_device() < 0:
                _lib.require_cuda(p)
            if p.dim() != 1 or not p.is_contiguous() or hidden not in (None, p.shape[0]):
                raise ValueError("weight and bias must be contiguous one-dimensional tensors of one length")
            if dtype not in (None, p.dtype):
                raise TypeError("weight and bias must share a dtype")
            if index not in (None, p.get_device()):
                raise RuntimeError("all tensors must share a device")
            hidden, index, dtype, code = p.shape[0], p.get_device(), p.dtype, _lib.dtype_code(p.dtype)
        weight_ptr, bias_ptr = _lib.ptr(weight), _lib.ptr(bias)
        params = _lib.NormParams(weight_ptr, bias_ptr, code, *self._constants)
        self._bound = bound = weight_ptr, bias_ptr, dtype, hidden, index, ctypes.byref(params)
        return bound

    @property
    def hidden(self) -> int | None:
        """The length of the weight and the bias; None without either."""
        return next((p.shape[0] for p in (self.weight, self.bias) if p is not None), None)

    @property
    def kind(self) -> str:
        return next(name for name, code in KINDS.items() if code == self._constants[0])

    @property
    def eps(self) -> float:
        return self._bound[5]._obj.eps

    @property
    def weight_offset(self) -> float:
        return self._bound[5]._obj.weight_offset

    def _for(self, hidden: int, index: int):
        """The norm as a C argument for rows of `hidden` values on a device, after its checks against them."""
        # A module may have replaced its parameters' data (``p.data = ...``, ``module.to(...)``), a user the parameters
        # themselves; an address has one device.
        weight_ptr, bias_ptr, dtype, length, device, ref = self._bound
        weight, bias = self.weight, self.bias
        if weight is None:
            same = weight_ptr is None
        else:
            if weight.requires_grad or _forward_ad._current_level >= 0:
                _lib.refuse_grad("BlockNorm", weight)
            same = (weight.data_ptr() == weight_ptr and weight.dtype is dtype and weight.numel() == length
                    and weight.is_contiguous())
        if bias is None:
            same = same and bias_ptr is None
        else:
            if bias.requires_grad or _forward_ad._current_level >= 0:
                _lib.refuse_grad("BlockNorm", bias)
            same = (same and bias.data_ptr() == bias_ptr and bias.dtype is dtype and bias.numel() == length
                    and bias.is_contiguous())
        if not same:
            _, _, _, length, device, ref = self._bind()
        if length is not None:
            if length != hidden:
                raise ValueError(f"the norm has {length} weights, its input {hidden} values a row")
            if device != index:
                raise RuntimeError("all tensors must share a device")
        return ref

    def __call__(self, x: torch.Tensor, *, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                 quantize: bool = False):
        """The normed rows of x [..., hidden]: a tensor like x (in out_dtype when given), or with
        ``quantize=True`` a pair (int8 [T, hidden] with rows padded to 16 bytes, fp32 scales [T]).
        ``out`` may be x itself."""
        return _run_norm(x, self, out, out_dtype, quantize)


def _run_norm(x, norm, out, out_dtype, quantize):
    index = x.get_device()
    if index < 0:
        _lib.require_cuda(x)
    shape = x.shape
    hidden = shape[-1] if shape else 0
    if not 0 < hidden <= MAX_HIDDEN:
        _check_hidden(x, "x", MAX_HIDDEN if norm is not None else MAX_QUANTIZED)
    code = _lib.dtype_code(x.dtype)
    if x.requires_grad or _forward_ad._current_level >= 0:
        _lib.refuse_grad("quantize_rows" if norm is None else "BlockNorm", x)
    norm_ref = None if norm is None else norm._for(hidden, index)
    rows, ld = _rows(x)
    t = x.numel() // hidden
    if t > MAX_ROWS:
        raise ValueError(f"x has {t} rows: at most {MAX_ROWS}")
    scale, ld_out = None, hidden
    if quantize:
        if out is not None or out_dtype is not None:
            raise ValueError("quantize=True returns its own int8 rows: out and out_dtype do not apply")
        out = int8_rows(t, hidden, x.device)
        ld_out += -hidden % 16
        scale = torch.empty(t, dtype=torch.float32, device=x.device)
        out_code = _lib.DTYPE_I8
    elif out is None:
        if out_dtype is None or out_dtype == x.dtype:
            out_code = code
            out = torch.empty_like(rows) if rows is x else x.new_empty(shape)
        else:
            out_code = _lib.dtype_code(out_dtype)
            out = torch.empty(shape, dtype=out_dtype, device=x.device)
    else:
        out_dtype = out_dtype or out.dtype
        out_code = _lib.dtype_code(out_dtype)
        ld_out = _out_rows(out, shape, t, out_dtype, index, "out")
        _check_overlap(_extent(out, ld_out, hidden, t), "out", (("x", _extent(rows, ld, hidden, t)),))
    lib = _lib.library()
    args = (rows.data_ptr(), ld, code, t, hidden, norm_ref, out.data_ptr(), ld_out, out_code,
            None if scale is None else scale.data_ptr())
    fn = lib.qcc_norm_rows
    status = fn(*args, _raw_stream(index)) if _current_device() == index else _lib.launch(index, fn, *args)
    if status:
        _lib.check(status, "qcc_norm_rows")
    return (out, scale) if quantize else out


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., cols] in bf16 / fp16 / fp32 -> (int8 [T, cols], fp32 scales [T]), one symmetric scale a row.

    scale = amax / 127 and q = round_half_even(127 * x / amax), of the exact quotient.  A row with
    amax < 2^-119 gets scale 0 and zeros; one that holds a NaN or an infinity
    gets scale NaN and zeros, so every product with it is NaN.  The int8 rows
    start on multiples of 16 bytes, as ``runtime.int8_dense`` wants them.  At
    most 131071 columns (rows beyond 32768 read their values twice).
    """
    return _run_norm(x, None, None, None, True)


def _gate_params(gate: torch.Tensor, activation: str | None, shape: torch.Size):
    """(gate rows, kept alive for the call; the gate as a C argument): rows of 1 or hidden values, each used by
    consecutive rows of the branch."""
    code = _lib.dtype_code(gate.dtype)
    cols = gate.shape[-1] if gate.dim() else 1
    if cols != 1 and cols != shape[-1] or gate.dim() > len(shape):
        raise ValueError(f"gate {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
    each = 1
    if gate.shape[:-1] != shape[:-1]:
        # Rows shared by the trailing leading axes (per sequence, or one row for all), full before them.
        lead, x_lead = list(gate.shape[:-1]), list(shape[:-1])
        lead = [1] * (len(x_lead) - len(lead)) + lead
        while lead and lead[-1] == 1:
            lead.pop()
            each *= x_lead[len(lead)]
        if lead != x_lead[:len(lead)]:
            raise ValueError(f"gate {tuple(gate.shape)} does not broadcast to {tuple(shape)} along its last axes")
    rows = gate if gate.dim() == 2 else gate.reshape(-1, cols)
    if rows.stride(1) != 1 and cols != 1:
        rows = rows.contiguous()
    return rows, ctypes.byref(_lib.GateParams(rows.data_ptr(), rows.stride(0), max(each, 1), cols, code,
                                              GATES[activation]))


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
    ``quantize=True``.  An output may be branch or residual itself
    (``residual_out=residual, out=branch`` run in place); other overlaps are
    refused.
    """
    index = branch.get_device()
    if index < 0 or residual.get_device() != index or (gate is not None and gate.get_device() != index):
        _lib.require_cuda(branch, residual, gate)
    shape = branch.shape
    if residual.shape != shape:
        raise ValueError(f"residual {tuple(residual.shape)} must have branch's shape {tuple(shape)}")
    hidden = shape[-1] if shape else 0
    if not 0 < hidden <= MAX_HIDDEN:
        _check_hidden(branch, "branch")
    code, res_code = _lib.dtype_code(branch.dtype), _lib.dtype_code(residual.dtype)
    if res_code != code and res_code != _lib.DTYPE_F32:
        raise TypeError("residual must be in branch's dtype or float32")
    if gate_activation not in GATES:
        raise ValueError(f"gate_activation must be one of {tuple(GATES)}")
    if next_norm is None and (quantize or out is not None or out_dtype is not None):
        raise ValueError("quantize, out and out_dtype need a next_norm")
    if (branch.requires_grad or residual.requires_grad or (gate is not None and gate.requires_grad)
            or _forward_ad._current_level >= 0):
        _lib.refuse_grad("residual_norm", branch, residual, gate)
    post_ref = None if post is None else post._for(hidden, index)
    next_ref = None if next_norm is None else next_norm._for(hidden, index)
    gate_rows, gate_ref = (None, None) if gate is None else _gate_params(gate, gate_activation, shape)
    rows, ld = _rows(branch)
    res_rows, ld_res = _rows(residual)
    t = branch.numel() // hidden
    if t > MAX_ROWS:
        raise ValueError(f"branch has {t} rows: at most {MAX_ROWS}")
    given = out is not None
    if residual_out is None:
        residual_out = torch.empty_like(residual) if res_rows is residual else residual.new_empty(shape)
        ld_res_out = hidden
    else:
        ld_res_out = _out_rows(residual_out, shape, t, residual.dtype, index, "residual_out")
        given = True
    scale_ptr, out_ptr, ld_out, out_code = None, None, hidden, code
    if next_norm is not None:
        if quantize:
            if out is not None or out_dtype is not None:
                raise ValueError("quantize=True returns its own int8 rows: out and out_dtype do not apply")
            out = int8_rows(t, hidden, branch.device)
            ld_out += -hidden % 16
            scale = torch.empty(t, dtype=torch.float32, device=branch.device)
            scale_ptr, out_code = scale.data_ptr(), _lib.DTYPE_I8
        elif out is None:
            if out_dtype is None or out_dtype == branch.dtype:
                out = torch.empty_like(rows) if rows is branch else branch.new_empty(shape)
            else:
                out_code = _lib.dtype_code(out_dtype)
                out = torch.empty(shape, dtype=out_dtype, device=branch.device)
        else:
            out_dtype = out_dtype or out.dtype
            out_code = _lib.dtype_code(out_dtype)
            ld_out = _out_rows(out, shape, t, out_dtype, index, "out")
        out_ptr = out.data_ptr()
    if given:
        branch_extent, res_extent = _extent(rows, ld, hidden, t), _extent(res_rows, ld_res, hidden, t)
        r_extent = res_extent if residual_out is res_rows else _extent(residual_out, ld_res_out, hidden, t)
        x_extent = branch_extent if out is rows else None if out is None else _extent(out, ld_out, hidden, t)
        if x_extent is not None and _overlap(x_extent, r_extent):
            raise ValueError("out overlaps residual_out")
        if r_extent is not res_extent or x_extent is not branch_extent:  # else that was the one test that is left
            inputs = ("branch", branch_extent), ("residual", res_extent)
            _check_overlap(r_extent, "residual_out", inputs)
            if x_extent is not None:
                _check_overlap(x_extent, "out", inputs)
        if gate is not None:
            g_extent = _extent(gate_rows, max(gate_rows.stride(0), 1), gate_rows.shape[1], gate_rows.shape[0])
            for name, extent in (("residual_out", r_extent), ("out", x_extent)):
                if extent is not None and _overlap(extent, g_extent):
                    raise ValueError(f"{name} overlaps the gate")
    lib = _lib.library()
    args = (rows.data_ptr(), ld, code, res_rows.data_ptr(), ld_res, res_code, t, hidden, post_ref, gate_ref,
            residual_scale, branch_scale, residual_out.data_ptr(), ld_res_out, next_ref, out_ptr, ld_out, out_code,
            scale_ptr)
    fn = lib.qcc_residual_norm
    status = fn(*args, _raw_stream(index)) if _current_device() == index else _lib.launch(index, fn, *args)
    if status:
        _lib.check(status, "qcc_residual_norm")
    if next_norm is None:
        return residual_out
    return residual_out, ((out, scale) if quantize else out)
