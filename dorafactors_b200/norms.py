"""Layer norm and RMS norm with native forward and backward kernels.

``layer_norm`` and ``rms_norm`` are differentiable functions over the last
dimension; ``LayerNorm`` and ``RMSNorm`` are the modules (same parameter names as
``torch.nn``'s, so checkpoints load).  ``*_forward`` / ``*_backward`` are the two
passes for a program that keeps the statistics itself.

Statistics and sums are fp32 whatever the activations' type and each output is
rounded once.  The weight's and bias's gradients are summed in a fixed order,
so they do not change from run to run.  Activations are fp32, fp16 or bf16;
weight and bias are in the activations' type or fp32 (another type is converted
to fp32, its gradient back).  There is no CPU path.
"""

from __future__ import annotations

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _native


def _params(x, cols: int, weight, bias, what: str):
    """Checked operands: (weight, bias, their dtype code)."""
    if not x.is_cuda:
        _native.require_cuda(x, what=what)
    act = _native.DTYPE_CODE.get(x.dtype)
    if act is None:
        _native.dtype_code(x)
    dtype = None
    for v, name in ((weight, "weight"), (bias, "bias")):
        if v is not None:
            if v.shape != (cols,):
                raise ValueError(f"{what}: {name} {tuple(v.shape)} does not match the last dimension {cols}")
            if v.get_device() != x.get_device():
                _native.require_cuda(x, v, what=what)
            dtype = v.dtype if dtype in (None, v.dtype) else torch.float32
    if dtype is None:
        return None, None, act
    if dtype is not x.dtype:
        dtype = torch.float32
    if weight is not None and not (weight.dtype is dtype and weight.is_contiguous()):
        weight = weight.to(dtype).contiguous()
    if bias is not None and not (bias.dtype is dtype and bias.is_contiguous()):
        bias = bias.to(dtype).contiguous()
    return weight, bias, _native.DTYPE_CODE[dtype]


def _forward(x, weight, bias, eps, rms: bool, what: str):
    shape = x.shape
    if not shape:
        raise ValueError(f"{what}: the input must have at least one dimension")
    if not eps >= 0:
        raise ValueError(f"{what}: eps must not be negative, got {eps}")
    w, b, code = _params(x, shape[-1], weight, bias, what)
    data, rows, cols, ld = _native.rows_of(x)
    y = torch.empty_like(x) if data is x and ld == cols else x.new_empty(shape)
    lead = shape[:-1]
    rstd = x.new_empty(lead, dtype=torch.float32)
    mean = None if rms else x.new_empty(lead, dtype=torch.float32)
    if rows and cols:
        _native.layer_norm_fwd(data, rows, cols, ld, w, b, code, eps, y, mean, rstd, rms)
    return y, mean, rstd


def _backward(dy, x, weight, mean, rstd, need, rms: bool, what: str, bias_dtype=None):
    if not x.ndim:
        raise ValueError(f"{what}: the input must have at least one dimension")
    w, _, code = _params(x, x.shape[-1], weight, None, what)
    if dy.shape != x.shape:
        raise ValueError(f"{what}: dy {tuple(dy.shape)} and x {tuple(x.shape)} differ in shape")
    _native.require_cuda(x, dy, mean, rstd, what=what)
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t is None and name == "mean" and rms:
            continue
        if t.dtype is not torch.float32 or t.numel() != x.shape[:-1].numel() or not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be the contiguous fp32 tensor {tuple(x.shape[:-1])} of the forward pass")
    if dy.dtype is not x.dtype:
        dy = dy.to(x.dtype)
    wdt = torch.float32 if code == 0 else x.dtype
    data, rows, cols, ldx = _native.rows_of(x)
    grad, _, _, lddy = _native.rows_of(dy)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
    dw = torch.empty(cols, dtype=wdt, device=x.device) if need[1] else None
    db = torch.empty(cols, dtype=wdt, device=x.device) if need[2] else None
    if cols and (need[0] or need[1] or need[2]):
        _native.layer_norm_bwd(grad, lddy, data, ldx, rows, cols, w, code, mean, rstd, dx, dw, db, rms)
    if dw is not None and weight is not None and dw.dtype is not weight.dtype:
        dw = dw.to(weight.dtype)
    if db is not None and bias_dtype is not None and db.dtype is not bias_dtype:
        db = db.to(bias_dtype)
    return dx, dw, db


def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5):
    """``(y, mean, rstd)``: y in x's shape and type, the fp32 statistics in its leading shape."""
    return _forward(x, weight, bias, eps, False, "layer_norm_forward")


def rms_norm_forward(x, weight=None, eps: float = 1e-6):
    """``(y, rstd)`` of the RMS norm."""
    y, _, rstd = _forward(x, weight, None, eps, True, "rms_norm_forward")
    return y, rstd


def layer_norm_backward(dy, x, weight, mean, rstd, need=(True, True, True)):
    """``(dx, d_weight, d_bias)``; those that ``need`` excludes are None.  The vectors are
    in ``weight``'s type (the activations' where weight is None)."""
    return _backward(dy, x, weight, mean, rstd, need, False, "layer_norm_backward",
                     None if weight is None else weight.dtype)


def rms_norm_backward(dy, x, weight, rstd, need=(True, True)):
    """``(dx, d_weight)`` of the RMS norm."""
    return _backward(dy, x, weight, None, rstd, (need[0], need[1], False), True, "rms_norm_backward")[:2]


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, rms):
        y, mean, rstd = _forward(x, weight, bias, eps, rms, "rms_norm" if rms else "layer_norm")
        ctx.rms = rms
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(x, weight, rstd, *(() if rms else (mean,)))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, rstd, *mean = ctx.saved_tensors
        need = (ctx.needs_input_grad[0], weight is not None and ctx.needs_input_grad[1],
                ctx.bias_dtype is not None and ctx.needs_input_grad[2])
        dx, dw, db = _backward(dy, x, weight, mean[0] if mean else None, rstd, need, ctx.rms,
                               "rms_norm backward" if ctx.rms else "layer_norm backward", ctx.bias_dtype)
        return dx, dw, db, None, None


def _tracked(x, weight, bias) -> bool:
    return x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension."""
    if torch.is_grad_enabled() and _tracked(x, weight, bias):
        return _Norm.apply(x, weight, bias, eps, False)
    return _forward(x, weight, bias, eps, False, "layer_norm")[0]


def rms_norm(x, weight=None, eps: float = 1e-6) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension."""
    if torch.is_grad_enabled() and _tracked(x, weight, None):
        return _Norm.apply(x, weight, None, eps, True)
    return _forward(x, weight, None, eps, True, "rms_norm")[0]


class LayerNorm(nn.Module):
    """``layer_norm`` over a last dimension of ``dim``."""

    def __init__(self, dim: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None,
                 dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(dim, device=device, dtype=dtype)) if elementwise_affine and bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps)


class RMSNorm(nn.Module):
    """``rms_norm`` over a last dimension of ``dim``."""

    def __init__(self, dim: int, eps: float = 1e-6, elementwise_affine: bool = True, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim, device=device, dtype=dtype)) if elementwise_affine else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return rms_norm(x, self.weight, self.eps)
