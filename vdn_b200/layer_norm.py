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

__all__ = ["layer_norm", "layer_norm_backward"]

@functools.lru_cache(maxsize=1024)
def _workspace_size(rows, width):
    return _lib.load().vdn_layer_norm_backward_workspace_size(rows, width)


def _rows(t, width):
    """(t as rows of unit column stride, a view where the layout allows it; rows; row stride)"""
    if t.is_contiguous():
        return t, t.numel() // width, width
    flat = t.reshape(-1, width)
    if flat.stride(1) != 1 and width != 1:
        flat = flat.contiguous()
    return flat, flat.shape[0], flat.stride(0) if flat.shape[0] > 1 else width


def _check(x, weight, bias):
    """(device index, width, x's dtype code, the parameters' dtype code) of valid arguments."""
    code = _lib.DTYPE_CODES.get(x.dtype) if isinstance(x, torch.Tensor) else None
    if code is None:
        raise TypeError("x must be an fp32, bf16 or fp16 tensor")
    index = x.get_device()
    if index < 0:
        raise ValueError("x must be a CUDA tensor")
    index = _lib.device_index(x, "x")
    width = x.shape[-1] if x.dim() else 0
    if width < 1:
        raise ValueError("x must have a last dimension to normalise")
    w_code = None
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        kind = _lib.DTYPE_CODES.get(t.dtype)
        if kind != code and kind != _lib.DTYPE_F32:
            raise TypeError(f"{name} must be {x.dtype} or fp32, got {t.dtype}")
        if t.dim() != 1 or t.numel() != width or t.get_device() != index:
            raise ValueError(f"{name} must be [{width}] on x's device")
        if w_code is not None and kind != w_code:
            raise TypeError("weight and bias must share one dtype")
        w_code = kind
    return index, width, code, code if w_code is None else w_code


def _like(t):
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _forward(x, weight, bias, eps, stats):
    _lib.refuse_tangents("layer_norm", x, weight, bias)
    index, width, code, w_code = _check(x, weight, bias)
    flat, rows, ld = _rows(x, width)
    y = _like(x)
    mean = rstd = w = b = None
    if stats:
        mean, rstd = torch.empty(2, rows, dtype=torch.float32, device=x.device)
    if weight is not None:
        w = weight if weight.is_contiguous() else weight.contiguous()
    if bias is not None:
        b = bias if bias.is_contiguous() else bias.contiguous()
    _lib.call_on(index, "vdn_layer_norm", flat.data_ptr(), code, rows, width, ld, w.data_ptr() if w is not None else None,
                 b.data_ptr() if b is not None else None, w_code, eps, y.data_ptr(), width,
                 mean.data_ptr() if stats else None, rstd.data_ptr() if stats else None)
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
    _lib.refuse_tangents("layer_norm_backward", grad_y, x, weight, mean, rstd)
    index, width, code, kind = _check(x, weight, None)
    if grad_y.shape != x.shape or grad_y.dtype != x.dtype or grad_y.get_device() != index:
        raise ValueError("grad_y must match x in shape, dtype and device")
    (flat, rows, x_ld), (dy, _, dy_ld) = _rows(x, width), _rows(grad_y, width)
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if t.dtype != torch.float32 or t.dim() != 1 or t.numel() != rows or t.get_device() != index:
            raise ValueError(f"{name} must be fp32 [{rows}] on x's device")
    device, dtype = x.device, x.dtype if weight is None else weight.dtype
    if weight is None and bias_dtype is not None:
        dtype, kind = bias_dtype, _lib.dtype_code(bias_dtype)
    dx = _like(x)
    dw = torch.empty(width, dtype=dtype, device=device) if want_w else None
    db = torch.empty(width, dtype=dtype, device=device) if want_b else None
    need = _workspace_size(rows, width)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    w = None if weight is None else weight.contiguous()
    mean, rstd = mean.contiguous(), rstd.contiguous()
    _lib.call_on(index, "vdn_layer_norm_backward", dy.data_ptr(), code, rows, width, dy_ld, flat.data_ptr(), x_ld,
                 None if w is None else w.data_ptr(), kind, mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), width,
                 dw.data_ptr() if want_w else None, db.data_ptr() if want_b else None, ws.data_ptr(), need,
                 _lib.status_word(index))
    return dx, dw, db


def layer_norm_backward(grad_y, x, weight, mean, rstd, *, bias=True):
    """(grad of x, of weight, of bias) from the forward's statistics; the weight's is None
    where there is no weight, the bias's unless `bias`.  Parameter gradients come in the
    weight's dtype (x's without one), summed over the rows in fp32 in a fixed order.
    Records nothing for autograd."""
    return _backward(grad_y, x, weight, mean, rstd, weight is not None, bool(bias))
