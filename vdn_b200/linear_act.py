"""Linear layer with bias, activation and residual in one kernel, with its gradients.

    y = act(x @ weight.T + bias) + residual        act: none, gelu_tanh, gelu_erf, silu

in bf16 or fp16 on tcgen05 with fp32 accumulation (vdn_linear_act): the trainable 16-bit
counterpart of the block's MXFP8 projections and their fused epilogues
(src/models/ops/mxfp8_linear.py:60-102).  The activation and the residual add work on the
fp32 sum; y is rounded once.

Differentiable: with gradients enabled, linear_act records itself for autograd; the same
backward is public as linear_act_backward (the form to capture into a CUDA graph).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["linear_act", "linear_act_backward", "ACTIVATIONS"]

ACTIVATIONS = {"none": _lib.ACT_NONE, "gelu_tanh": _lib.ACT_GELU_TANH, "gelu_erf": _lib.ACT_GELU_ERF,
               "silu": _lib.ACT_SILU}


def _matrix(t, cols):
    """t [..., cols] as (rows of unit column stride, their count, their stride)."""
    if t.is_contiguous():
        return t, t.numel() // cols, cols
    flat = t.reshape(-1, cols)
    ld = flat.stride(0)
    if (flat.stride(1) != 1 and cols != 1) or (ld < cols and flat.shape[0] > 1):
        flat, ld = flat.contiguous(), cols
    return flat, flat.shape[0], max(ld, cols)


def _check(x, weight, act):
    """(device index, dtype code) of valid arguments."""
    if not isinstance(x, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("x and weight must be tensors")
    dtype = x.dtype
    if (dtype != torch.bfloat16 and dtype != torch.float16) or weight.dtype != dtype:
        raise TypeError(f"x and weight must both be bf16 or both fp16, got {x.dtype} and {weight.dtype}")
    index = x.get_device()
    if index < 0 or weight.get_device() != index:
        raise ValueError("x and weight must be CUDA tensors on one device")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError("x must be [..., k] and weight [n, k]")
    if weight.numel() < 1:
        raise ValueError("weight must not be empty")
    if act not in ACTIVATIONS:
        raise ValueError(f"act must be one of {tuple(ACTIVATIONS)}, got {act!r}")
    return _lib.device_index(x, "x"), _lib.DTYPE_CODES[dtype]


def _same(t, x, index, shape, name):
    if t.dtype != x.dtype or t.get_device() != index:
        raise TypeError(f"{name} must have x's dtype and device")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")


def _forward(x, weight, bias, act, residual, want_pre):
    _lib.refuse_tangents("linear_act", x, weight, bias, residual)
    index, code = _check(x, weight, act)
    n, k = weight.shape
    shape = (*x.shape[:-1], n)
    device = x.device
    res = pre = ws = None
    ldr = need = 0
    if bias is not None:
        _same(bias, x, index, (n,), "bias")
        bias = bias if bias.is_contiguous() else bias.contiguous()
    if residual is not None:
        _same(residual, x, index, shape, "residual")
        res, _, ldr = _matrix(residual, n)
    flat, rows, ldx = _matrix(x, k)
    w, _, ldw = _matrix(weight, k)
    y = torch.empty(shape, dtype=x.dtype, device=device)
    if want_pre:
        pre = torch.empty(shape, dtype=x.dtype, device=device)
    px, pw = flat.data_ptr(), w.data_ptr()
    if ldx % 8 or ldw % 8 or px % 16 or pw % 16:     # rows the tensor maps do not take: room for copies
        need = _lib.load().vdn_linear_workspace_size(px, ldx, pw, ldw, rows, n, k)
        ws = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.call_on(index, "vdn_linear_act", px, ldx, pw, ldw, None if bias is None else bias.data_ptr(),
                 None if res is None else res.data_ptr(), ldr, code, ACTIVATIONS[act], rows, n, k, y.data_ptr(), n,
                 None if pre is None else pre.data_ptr(), n, None if ws is None else ws.data_ptr(), need,
                 _lib.status_word(index))
    return y, pre


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, act, residual):
        y, pre = _forward(x, weight, bias, act, residual, act != "none")
        ctx.save_for_backward(x, weight, pre)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        _lib.refuse_captured_autograd("linear_act", ctx.saved_tensors[0])
        x, weight, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db = _backward(grad_y, x, weight, pre, ctx.act, need[0], need[1], need[2])
        return dx, dw, db, None, grad_y if need[4] else None


def linear_act(x, weight, bias=None, *, act="none", residual=None, return_pre=False):
    """act(x @ weight.T + bias) + residual for x [..., k], weight [n, k], bias [n] and residual
    [..., n], all bf16 or all fp16; act is one of ACTIVATIONS.  With return_pre also
    x @ weight.T + bias, rounded (what linear_act_backward takes for an activation).

    Row-strided operands are read in place where their rows are 16-byte aligned; the
    library copies others (odd k, offset views) into padded rows first."""
    if torch.is_grad_enabled() and _lib.records(x, weight, bias, residual):
        if return_pre:
            raise ValueError("return_pre is for the explicit backward, not where gradients are recorded")
        _lib.refuse_captured_autograd("linear_act", x)
        return _LinearAct.apply(x, weight, bias, act, residual)
    y, pre = _forward(x, weight, bias, act, residual, return_pre)
    return (y, pre) if return_pre else y


def _backward(grad_y, x, weight, pre, act, want_x, want_w, want_b):
    _lib.refuse_tangents("linear_act_backward", grad_y, x, weight, pre)
    index, dtype = _check(x, weight, act)
    n, k = weight.shape
    shape = (*x.shape[:-1], n)
    _same(grad_y, x, index, shape, "grad_y")
    z, ldp = None, 0
    if act != "none":
        if pre is None:
            raise ValueError("pre (linear_act's return_pre) is needed for the activation's gradient")
        _same(pre, x, index, shape, "pre")
        z, _, ldp = _matrix(pre, n)
    dev, code = x.device, ACTIVATIONS[act]
    dy, rows, ldy = _matrix(grad_y, n)
    flat, _, ldx = _matrix(x, k)
    w, _, ldw = _matrix(weight, k)
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_x else None
    dw = torch.empty(n, k, dtype=x.dtype, device=dev) if want_w else None
    db = torch.empty(n, dtype=x.dtype, device=dev) if want_b else None
    pdy, px, pw = dy.data_ptr(), flat.data_ptr(), w.data_ptr()
    need = _lib.load().vdn_linear_backward_workspace_size(pdy, ldy, px, ldx, pw, ldw, code, rows, n, k)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _lib.call_on(index, "vdn_linear_act_backward", pdy, ldy, None if z is None else z.data_ptr(), ldp, px, ldx, pw, ldw,
                 dtype, code, rows, n, k, dx.data_ptr() if want_x else None, k, dw.data_ptr() if want_w else None, k,
                 db.data_ptr() if want_b else None, ws.data_ptr(), need, _lib.status_word(index))
    return dx, dw, db


def linear_act_backward(grad_y, x, weight, pre=None, *, act="none", bias=True):
    """(grad of x, of weight, of bias or None) from the forward's inputs and `pre`.  The residual's
    gradient is grad_y.  The activation's gradient enters the two products rounded to the
    operands' type (in fp16 it is infinite above 65504, which takes a grad_y near that limit: the
    slopes stay below 1.13); the bias gradient sums it unrounded, in fp32 and a fixed order.  Records
    nothing for autograd."""
    return _backward(grad_y, x, weight, pre, act, True, True, bool(bias))
