"""Gated linear recurrence per channel and token, with its gradients (vdn_gated_scan).

    h_t = exp(log_decay_t) * h_{t-1} + x_t,    y_t = h_t

the diagonal companion of the frame-wise delta-rule scans of the VDA branch
(src/models/linear_attention/scan.py:270-355): it runs over tokens, takes batches or
packed sequences, either direction and an initial state, and has a backward pass.  One
token per sequence is the serving step: pass `state` and reuse it as `out_state`.

Differentiable: with gradients enabled, gated_scan records itself for autograd; the same
backward is public as gated_scan_backward (the form to capture into a CUDA graph).
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .mxfp8_linear import _status

__all__ = ["gated_scan", "gated_scan_backward"]

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _layout(x, log_decay, state, cu_seqlens, what):
    """(lead dims, sequences, rows, heads, head dim, shared decay) after the argument checks."""
    if not isinstance(x, torch.Tensor) or not isinstance(log_decay, torch.Tensor):
        raise TypeError(f"{what} and log_decay must be tensors")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what} must be fp32, bf16 or fp16, got {x.dtype}")
    if log_decay.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"log_decay must be {x.dtype} or fp32, got {log_decay.dtype}")
    if not x.is_cuda or log_decay.device != x.device:
        raise ValueError(f"{what} and log_decay must be CUDA tensors on one device")
    _lib.require_device(x, what)
    lead = 2 if cu_seqlens is None else 1
    if x.dim() - lead not in (1, 2):
        raise ValueError(f"{what} must be [B, T, C] or [B, T, H, d] (packed: [N, C] or [N, H, d])")
    tail = x.shape[lead:]
    heads, d = (tail[0], tail[1]) if len(tail) == 2 else (1, tail[0])
    shared = log_decay.dim() == lead + 1 and len(tail) == 2
    if log_decay.shape != (x.shape[:-1] if shared else x.shape):
        raise ValueError(f"log_decay must have {what}'s shape, or one value per head of [.., H, d]")
    if shared and d not in (32, 64, 128):
        raise ValueError("a decay per head needs a head dim of 32, 64 or 128 (expand it per channel for others)")
    if cu_seqlens is None:
        seqs, rows = x.shape[:2]
    else:
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.device != x.device:
            raise ValueError("cu_seqlens must be int32 [sequences + 1] on the device of the rows")
        if cu_seqlens.numel() < 1 or not cu_seqlens.is_contiguous():
            raise ValueError("cu_seqlens must be contiguous and hold at least one offset")
        seqs, rows = cu_seqlens.numel() - 1, x.shape[0]
    _check_state(state, x, (seqs, *tail), "state")
    return lead, seqs, rows, heads, d, shared


def _check_state(state, x, shape, name):
    if state is None:
        return
    if state.dtype != torch.float32 or state.device != x.device:
        raise TypeError(f"{name} must be fp32 on the device of the rows")
    if state.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(state.shape)}")


def _flat(t, lead):
    """t with its trailing dims laid out as one contiguous row of channels (copied if not)."""
    size, stride = t.shape[lead:], t.stride()[lead:]
    need = 1
    for n, s in zip(reversed(size), reversed(stride)):
        if n != 1 and s != need:
            return t.contiguous()
        need *= n
    return t


def _strides(t, lead):
    """(batch stride, row stride); a stride that no index multiplies counts as 0."""
    row = t.stride(lead - 1) if t.shape[lead - 1] > 1 else 0
    return (t.stride(0) if t.shape[0] > 1 else 0) if lead == 2 else 0, row


def _output(out, x, lead, name):
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"{name} must match the rows in shape, dtype and device")
    if _flat(out, lead) is not out:
        raise ValueError(f"{name}'s channels must be contiguous")
    return out


def _forward(x, log_decay, state, cu_seqlens, reverse, out, out_state):
    lead, seqs, rows, heads, d, shared = _layout(x, log_decay, state, cu_seqlens, "x")
    y = _output(out, x, lead, "out")
    shape = (seqs, *x.shape[lead:])
    if out_state is None:
        out_state = torch.empty(shape, dtype=torch.float32, device=x.device)
    else:
        _check_state(out_state, x, shape, "out_state")
        if not out_state.is_contiguous():
            raise ValueError("out_state must be contiguous")
    if heads * d == 0:
        return y, out_state
    if seqs == 0:
        return (y.zero_() if out is None else y), out_state
    x, log_decay = _flat(x, lead), _flat(log_decay, lead)
    state = None if state is None else state.contiguous()
    _lib.call_on(x.device, "vdn_gated_scan", x.data_ptr(), _lib.dtype_code(x.dtype), *_strides(x, lead),
                 log_decay.data_ptr(), _lib.dtype_code(log_decay.dtype), *_strides(log_decay, lead), int(shared),
                 _lib.ptr(state), _lib.ptr(cu_seqlens), seqs, rows, heads, d, int(bool(reverse)), y.data_ptr(),
                 *_strides(y, lead), int(out is None), out_state.data_ptr(), _status(x.device).data_ptr())
    return y, out_state


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, log_decay, state, cu_seqlens, reverse):
        ctx.set_materialize_grads(False)
        y, last = _forward(x, log_decay, state, cu_seqlens, reverse, None, None)
        ctx.save_for_backward(log_decay, y, state, cu_seqlens)
        ctx.reverse = reverse
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y, grad_last):
        log_decay, y, state, cu_seqlens = ctx.saved_tensors
        if grad_y is None:
            grad_y = torch.zeros_like(y)
        dx, dg, ds = gated_scan_backward(grad_y, log_decay, y, state=state, grad_state=grad_last,
                                         cu_seqlens=cu_seqlens, reverse=ctx.reverse)
        return dx, dg, ds if state is not None else None, None, None


def gated_scan(x, log_decay, state=None, *, cu_seqlens=None, reverse=False, out=None, out_state=None):
    """y, last state of h_t = exp(log_decay_t) h_{t-1} + x_t.

    x [B, T, C] or [B, T, H, d] (fp32, bf16 or fp16); log_decay of x's shape, or [B, T, H]
    for one decay per head (d = 32, 64 or 128), in x's dtype or fp32; -inf restarts a
    channel.  With cu_seqlens (int32 [S + 1] on the device, nondecreasing row offsets) the
    sequences lie end to end: x [N, C] or [N, H, d]; rows behind the last offset come back
    zero, and stay as they were in a caller's `out`.  state / out_state fp32 [B or S, C] or
    [.., H, d]; out_state may be `state` (updated in place).  reverse runs each sequence from
    its last row to its first.  Strided rows and expanded log_decay are read in place as
    long as a row's channels are contiguous.  A state that overflows fp32 comes out as inf or NaN.
    """
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad
                                       for t in (x, log_decay, state)):
        if out is not None or out_state is not None:
            raise ValueError("out and out_state cannot be given where gradients are recorded")
        _lib.refuse_captured_autograd("gated_scan")
        return _GatedScan.apply(x, log_decay, state, cu_seqlens, bool(reverse))
    return _forward(x, log_decay, state, cu_seqlens, reverse, out, out_state)


@torch.no_grad()
def gated_scan_backward(grad_y, log_decay, y, *, state=None, grad_state=None, cu_seqlens=None, reverse=False):
    """(grad of x, of log_decay, of state) from the forward's output y and its arguments.

    grad_state is the gradient of the last state, if any; the gradient of the first state
    comes back as fp32 also when `state` was None.  Rows behind the last packed sequence
    have zero gradients."""
    lead, seqs, rows, heads, d, shared = _layout(y, log_decay, state, cu_seqlens, "y")
    if grad_y.shape != y.shape or grad_y.dtype != y.dtype or grad_y.device != y.device:
        raise ValueError("grad_y must match y in shape, dtype and device")
    shape = (seqs, *y.shape[lead:])
    _check_state(grad_state, y, shape, "grad_state")
    dx = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    dg = torch.empty(log_decay.shape, dtype=log_decay.dtype, device=y.device)
    ds = torch.empty(shape, dtype=torch.float32, device=y.device)
    if heads * d == 0 or seqs == 0:
        return dx.zero_(), dg.zero_(), ds
    grad_y, log_decay, y = _flat(grad_y, lead), _flat(log_decay, lead), _flat(y, lead)
    state = None if state is None else state.contiguous()
    grad_state = None if grad_state is None else grad_state.contiguous()
    _lib.call_on(y.device, "vdn_gated_scan_backward", grad_y.data_ptr(), _lib.dtype_code(y.dtype),
                 *_strides(grad_y, lead), log_decay.data_ptr(), _lib.dtype_code(log_decay.dtype),
                 *_strides(log_decay, lead), int(shared), y.data_ptr(), *_strides(y, lead), _lib.ptr(state),
                 _lib.ptr(grad_state), _lib.ptr(cu_seqlens), seqs, rows, heads, d, int(bool(reverse)),
                 dx.data_ptr(), *_strides(dx, lead), dg.data_ptr(), *_strides(dg, lead), 1, ds.data_ptr(),
                 _status(y.device).data_ptr())
    return dx, dg, ds
