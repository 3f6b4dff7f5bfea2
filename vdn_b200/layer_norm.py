"""Layer norm over the last dimension, with its gradients (vdn_layer_norm).

    y = (x - mean) / sqrt(var + eps) * weight + bias

in fp32 for fp32, bf16 and fp16 rows; weight and bias in the rows' dtype or fp32, either
optional.  The trainable counterpart of the block's inference norms (RMSNorm of
src/models/ops/rms_norm.py:23-32 and the pre-norm producer).

Differentiable: with gradients enabled, layer_norm records itself for autograd; the same
backward is public as layer_norm_backward (the form to capture into a CUDA graph).
"""
from __future__ import annotations

import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .mxfp8_linear import status_address

__all__ = ["layer_norm", "layer_norm_backward"]

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


@functools.lru_cache(maxsize=1024)
def _workspace_size(rows, width):
    return _lib.load().vdn_layer_norm_backward_workspace_size(rows, width)


def _rows(t):
    """(t as rows of unit column stride, a view where the layout allows it; rows; row stride)"""
    width = t.shape[-1]
    if t.is_contiguous():
        return t, t.numel() // width, width
    flat = t.reshape(-1, width)
    if flat.stride(1) != 1 and width != 1:
        flat = flat.contiguous()
    return flat, flat.shape[0], flat.stride(0) if flat.shape[0] > 1 else width


def _check(x, weight, bias):
    if not isinstance(x, torch.Tensor) or x.dtype not in _DTYPES:
        raise TypeError("x must be an fp32, bf16 or fp16 tensor")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension to normalise")
    _lib.require_device(x, "x")
    if weight is not None:
        _check_parameter(x, weight, "weight")
    if bias is not None:
        _check_parameter(x, bias, "bias")
        if weight is not None and weight.dtype != bias.dtype:
            raise TypeError("weight and bias must share one dtype")


def _check_parameter(x, t, name):
    if t.dtype != x.dtype and t.dtype != torch.float32:
        raise TypeError(f"{name} must be {x.dtype} or fp32, got {t.dtype}")
    if t.dim() != 1 or t.shape[0] != x.shape[-1] or t.device != x.device:
        raise ValueError(f"{name} must be [{x.shape[-1]}] on x's device")


def _forward(x, weight, bias, eps, stats):
    _check(x, weight, bias)
    flat, rows, ld = _rows(x)
    width = x.shape[-1]
    device, code = x.device, _lib.dtype_code(x.dtype)
    y = torch.empty(x.shape, dtype=x.dtype, device=device)
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty(2, rows, dtype=torch.float32, device=device)
    given = weight if weight is not None else bias
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    _lib.call_on(device, "vdn_layer_norm", flat.data_ptr(), code, rows, width, ld, _lib.address(w), _lib.address(b),
                 code if given is None else _lib.dtype_code(given.dtype), eps, y.data_ptr(), width,
                 _lib.address(mean), _lib.address(rstd))
    return y, mean, rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        _lib.refuse_captured_autograd("layer_norm", ctx.saved_tensors[0])
        x, weight, bias, mean, rstd = ctx.saved_tensors
        dx, dw, db = _backward(grad_y, x, weight, mean, rstd, ctx.needs_input_grad[1], ctx.needs_input_grad[2],
                               None if bias is None else bias.dtype)
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, return_stats=False):
    """y of x's shape and dtype; with return_stats also the rows' mean and 1 / sqrt(var + eps)
    (fp32 [rows], what layer_norm_backward takes)."""
    if torch.is_grad_enabled() and _lib.records(x, weight, bias):
        if return_stats:
            raise ValueError("return_stats is for the explicit backward, not where gradients are recorded")
        _lib.refuse_captured_autograd("layer_norm", x)
        return _LayerNorm.apply(x, weight, bias, float(eps))
    y, mean, rstd = _forward(x, weight, bias, eps, return_stats)
    return (y, mean, rstd) if return_stats else y


def _backward(grad_y, x, weight, mean, rstd, want_w, want_b, bias_dtype=None):
    _check(x, weight, None)
    if grad_y.shape != x.shape or grad_y.dtype != x.dtype or grad_y.device != x.device:
        raise ValueError("grad_y must match x in shape, dtype and device")
    (flat, rows, x_ld), (dy, _, dy_ld) = _rows(x), _rows(grad_y)
    width = x.shape[-1]
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t.shape != (rows,) or t.dtype != torch.float32 or t.device != x.device:
            raise ValueError(f"{name} must be fp32 [{rows}] on x's device")
    kind = weight.dtype if weight is not None else bias_dtype or x.dtype
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = torch.empty(width, dtype=kind, device=x.device) if want_w else None
    db = torch.empty(width, dtype=kind, device=x.device) if want_b else None
    need = _workspace_size(rows, width)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    w = None if weight is None else weight.contiguous()
    mean, rstd = mean.contiguous(), rstd.contiguous()
    _lib.call_on(x.device, "vdn_layer_norm_backward", dy.data_ptr(), _lib.dtype_code(x.dtype), rows, width, dy_ld,
                 flat.data_ptr(), x_ld, _lib.address(w), _lib.dtype_code(kind), mean.data_ptr(), rstd.data_ptr(),
                 dx.data_ptr(), width, _lib.address(dw), _lib.address(db), ws.data_ptr(), need,
                 status_address(x.device))
    return dx, dw, db


@torch.no_grad()
def layer_norm_backward(grad_y, x, weight, mean, rstd, *, bias=True):
    """(grad of x, of weight, of bias) from the forward's statistics; the weight's is None
    where there is no weight, the bias's unless `bias`.  Parameter gradients come in the
    weight's dtype (x's without one), summed over the rows in fp32 in a fixed order."""
    return _backward(grad_y, x, weight, mean, rstd, weight is not None, bool(bias))
