"""Calls of the block norms and the int8 products that are refused, checked without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

import conftest  # noqa: F401
from qcc_b200 import _lib
from qcc_b200.runtime.block import FFNBlock
from qcc_b200.runtime.block_norm import BlockNorm, quantize_rows, residual_norm
from qcc_b200.runtime.int8_dense import Int8GatedFFN, Int8GatedLinear, Int8Linear, int8_gated_linear, int8_linear

P = ctypes.c_void_p(64)
BF16, F32, I8 = _lib.DTYPE_BF16, _lib.DTYPE_F32, _lib.DTYPE_I8


def params(kind=_lib.NORM_RMS, weight=64, bias=None, dtype=BF16):
    return ctypes.byref(_lib.NormParams(weight, bias, dtype, kind, 0.0, 1e-6))


def norm_args(**changed):
    a = dict(x=P, ldx=64, dtype=BF16, rows=2, hidden=64, norm=params(), out=P, ld_out=64, out_dtype=BF16, scale=None,
             stream=None)
    assert set(changed) <= set(a)
    a.update(changed)
    return list(a.values())


@pytest.mark.parametrize("changed,status", [
    (dict(dtype=7), _lib.ERR_DTYPE), (dict(dtype=I8), _lib.ERR_DTYPE), (dict(out_dtype=9), _lib.ERR_DTYPE),
    (dict(norm=params(kind=5)), _lib.ERR_INVALID_ARGUMENT), (dict(norm=params(dtype=8)), _lib.ERR_INVALID_ARGUMENT),
    (dict(norm=params(kind=_lib.NORM_NONE)), _lib.ERR_INVALID_ARGUMENT), (dict(rows=-1), _lib.ERR_SHAPE),
    (dict(hidden=0), _lib.ERR_SHAPE), (dict(ldx=63), _lib.ERR_SHAPE), (dict(ld_out=63), _lib.ERR_SHAPE),
    (dict(hidden=32769, ldx=32769, ld_out=32769), _lib.ERR_UNSUPPORTED), (dict(x=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(out=None), _lib.ERR_INVALID_ARGUMENT), (dict(out_dtype=I8), _lib.ERR_INVALID_ARGUMENT),
    (dict(x=ctypes.c_void_p(65)), _lib.ERR_ALIGNMENT), (dict(out=ctypes.c_void_p(65)), _lib.ERR_ALIGNMENT),
    (dict(norm=params(weight=65)), _lib.ERR_ALIGNMENT), (dict(norm=params(bias=66, dtype=F32)), _lib.ERR_ALIGNMENT),
    (dict(out_dtype=I8, scale=ctypes.c_void_p(66)), _lib.ERR_ALIGNMENT),
    (dict(rows=0, x=None, out=None, norm=None), _lib.OK)])
def test_norm_rows_status(changed, status):
    assert _lib.library().qcc_norm_rows(*norm_args(**changed)) == status


def gate(values=64, ld=1, each=1, cols=1, dtype=BF16, act=0):
    return ctypes.byref(_lib.GateParams(values, ld, each, cols, dtype, act))


def join_args(**changed):
    a = dict(branch=P, ld_branch=64, dtype=BF16, residual=P, ld_residual=64, residual_dtype=BF16, rows=2, hidden=64,
             post=None, gate=None, rscale=1.0, bscale=1.0, residual_out=P, ld_residual_out=64, next=None, out=None,
             ld_out=0, out_dtype=BF16, scale=None, stream=None)
    assert set(changed) <= set(a)
    a.update(changed)
    return list(a.values())


@pytest.mark.parametrize("changed,status", [
    (dict(residual_dtype=_lib.DTYPE_F16), _lib.ERR_DTYPE), (dict(dtype=F32), _lib.ERR_DTYPE),
    (dict(post=params(kind=4)), _lib.ERR_INVALID_ARGUMENT), (dict(next=params(kind=-1)), _lib.ERR_INVALID_ARGUMENT),
    (dict(ld_residual=60), _lib.ERR_SHAPE), (dict(ld_residual_out=60), _lib.ERR_SHAPE),
    (dict(gate=gate(dtype=I8)), _lib.ERR_DTYPE), (dict(gate=gate(act=3)), _lib.ERR_INVALID_ARGUMENT),
    (dict(gate=gate(each=0)), _lib.ERR_SHAPE), (dict(gate=gate(cols=32)), _lib.ERR_SHAPE),
    (dict(gate=gate(ld=-1)), _lib.ERR_SHAPE), (dict(gate=gate(values=None)), _lib.ERR_INVALID_ARGUMENT),
    (dict(out=P, ld_out=60), _lib.ERR_SHAPE), (dict(gate=gate(values=65)), _lib.ERR_ALIGNMENT),
    (dict(residual=ctypes.c_void_p(65)), _lib.ERR_ALIGNMENT),
    (dict(residual_out=ctypes.c_void_p(65)), _lib.ERR_ALIGNMENT),
    (dict(out=P, ld_out=64, out_dtype=I8), _lib.ERR_INVALID_ARGUMENT), (dict(residual=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(residual_out=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(hidden=40000, ld_branch=40000, ld_residual=40000, ld_residual_out=40000), _lib.ERR_UNSUPPORTED),
    (dict(rows=0, branch=None, residual=None), _lib.OK)])
def test_residual_norm_status(changed, status):
    assert _lib.library().qcc_residual_norm(*join_args(**changed)) == status


def linear_args(**changed):
    a = dict(x=P, ldx=64, xs=P, w=P, ldw=64, ws=P, bias=None, bias_dtype=F32, tokens=2, channels=8, cols=64, y=P,
             ldy=8, y_dtype=BF16, stream=None)
    assert set(changed) <= set(a)
    a.update(changed)
    return a


@pytest.mark.parametrize("changed,status", [
    (dict(y_dtype=I8), _lib.ERR_DTYPE), (dict(tokens=-1), _lib.ERR_SHAPE), (dict(channels=0), _lib.ERR_SHAPE),
    (dict(cols=0), _lib.ERR_SHAPE), (dict(ldx=48), _lib.ERR_SHAPE), (dict(ldw=48), _lib.ERR_SHAPE),
    (dict(ldy=7), _lib.ERR_SHAPE), (dict(cols=131072, ldx=131072, ldw=131072), _lib.ERR_UNSUPPORTED),
    (dict(tokens=(1 << 20) + 1), _lib.ERR_UNSUPPORTED),
    (dict(channels=(1 << 19) + 1, ldy=1 << 20), _lib.ERR_UNSUPPORTED),
    (dict(x=None), _lib.ERR_INVALID_ARGUMENT), (dict(ws=None), _lib.ERR_INVALID_ARGUMENT),
    (dict(y=None), _lib.ERR_INVALID_ARGUMENT), (dict(ldx=72), _lib.ERR_ALIGNMENT), (dict(ldw=72), _lib.ERR_ALIGNMENT),
    (dict(x=ctypes.c_void_p(72)), _lib.ERR_ALIGNMENT), (dict(w=ctypes.c_void_p(72)), _lib.ERR_ALIGNMENT),
    (dict(xs=ctypes.c_void_p(66)), _lib.ERR_ALIGNMENT), (dict(ws=ctypes.c_void_p(65)), _lib.ERR_ALIGNMENT),
    (dict(y=ctypes.c_void_p(65)), _lib.ERR_ALIGNMENT),
    (dict(tokens=0, x=None, y=None), _lib.OK)])
def test_int8_linear_status(changed, status):
    lib = _lib.library()
    a = linear_args(**changed)
    assert lib.qcc_int8_linear(*a.values()) == status
    gated = {k: v for k, v in a.items() if k not in ("bias", "bias_dtype")}
    assert lib.qcc_int8_gated_linear(*gated.values()) == status
    if status == _lib.OK:
        a["bias"], a["bias_dtype"] = P, I8
        assert lib.qcc_int8_linear(*a.values()) == _lib.ERR_DTYPE


def test_no_cpu_fallback():
    x = torch.zeros(2, 64)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        BlockNorm()(x)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        BlockNorm(torch.ones(64))
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        quantize_rows(x)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        residual_norm(x, x)
    q, s = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2)
    for call in (lambda: int8_linear(q, s, q, s), lambda: int8_gated_linear(q, s, q, s), lambda: Int8Linear(q, s)):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            call()


def test_python_argument_errors():
    with pytest.raises(ValueError, match="next_norm"):
        FFNBlock(lambda x: x, BlockNorm(), quantize_next=True)
    with pytest.raises(ValueError, match="kind"):
        BlockNorm(kind="batch")
    with pytest.raises(ValueError, match="eps"):
        BlockNorm(eps=-1.0)
    with pytest.raises(ValueError, match="weight_offset"):
        BlockNorm(weight_offset=1.0)
    s = torch.zeros(2)
    q = torch.zeros(2, 64, dtype=torch.int8)
    for bad, scale in ((q[0], s), (q.float(), s), (q.t(), s), (q, s.double()), (q, s[:1]), (q[:, :60].contiguous(), s),
                       (torch.zeros(2, 72, dtype=torch.int8), s)):
        with pytest.raises(ValueError):
            int8_linear(bad, scale, q, s)
        with pytest.raises(ValueError):
            Int8Linear(bad, scale)
    with pytest.raises(ValueError, match="matri"):
        Int8GatedLinear.from_weights(torch.zeros(2, 3), torch.zeros(3, 2))
    with pytest.raises(ValueError, match="bias"):
        Int8GatedLinear.from_weight(torch.zeros(2, 3), torch.zeros(1))
    with pytest.raises(ValueError):
        Int8GatedFFN.from_weights(torch.zeros(2, 3), torch.zeros(2, 3), torch.zeros(2, 3))


@pytest.mark.gpu
def test_gpu_argument_errors():
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda")
    norm = BlockNorm(torch.ones(64, device="cuda"))
    for call in (lambda: norm(x[:, :32]), lambda: norm(x, out=x.float(), out_dtype=torch.float16),
                 lambda: norm(x, out=x[:1]), lambda: norm(x, out=x, quantize=True), lambda: norm(x[:, :0]),
                 lambda: BlockNorm()(torch.zeros(1, 32769, device="cuda")),
                 lambda: norm(x, out=torch.zeros(64, 2, dtype=torch.bfloat16, device="cuda").t()),
                 lambda: norm(x, out=torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda").expand(2, 64)),
                 lambda: residual_norm(x, x[:1]), lambda: residual_norm(x, x, gate=x[:, :3]),
                 lambda: residual_norm(x, x, gate=x[:1].expand(3, 64)), lambda: residual_norm(x, x, quantize=True),
                 lambda: residual_norm(x, x, gate=x, gate_activation="relu"),
                 lambda: residual_norm(x, x, out_dtype=torch.float32)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: norm(x.double()), lambda: norm(x, out_dtype=torch.float64),
                 lambda: residual_norm(x, x.half()), lambda: residual_norm(x.float(), x),
                 lambda: BlockNorm(torch.ones(4, device="cuda", dtype=torch.float64)),
                 lambda: BlockNorm(torch.ones(4, device="cuda"), torch.ones(4, device="cuda").half())):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        residual_norm(x, x, gate=torch.zeros(64))
    grad = x.float().requires_grad_()
    weight = torch.ones(64, device="cuda", requires_grad=True)
    for call in (lambda: norm(grad), lambda: BlockNorm(weight)(x), lambda: residual_norm(x, grad),
                 lambda: residual_norm(x, x, gate=weight)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad():
            call()
    q, s = quantize_rows(x)
    wide = torch.zeros(4, 128, dtype=torch.int8, device="cuda")
    for call in (lambda: int8_linear(q, s, wide, torch.zeros(4, device="cuda")),
                 lambda: int8_gated_linear(q, s, wide[:3, :64], torch.zeros(3, device="cuda")),
                 lambda: int8_linear(q, s, wide[:0, :64], s[:0]),
                 lambda: int8_linear(wide[:2, 8:72], s, wide[:, :64], torch.zeros(4, device="cuda")),
                 lambda: int8_linear(q, s, q, s, bias=torch.zeros(3, device="cuda")),
                 lambda: int8_linear(q, s, q, s, out=torch.zeros(2, 3, device="cuda")),
                 lambda: int8_linear(q, s, q, s, out=torch.zeros(2, 2, device="cuda"), out_dtype=torch.bfloat16),
                 lambda: Int8Linear(q, s)(x[:, :32]),
                 lambda: Int8GatedFFN(Int8GatedLinear(q, s), Int8Linear(q, s))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        int8_linear(q, s, q, s, out_dtype=torch.float64)
