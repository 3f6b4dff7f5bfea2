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

__all__ = ["gated_scan", "gated_scan_backward"]

def _layout(x, log_decay, state, cu_seqlens, what):
    """(device index, dtype codes, lead dims, sequences, rows, heads, head dim, shared decay,
    state shape) after the argument checks."""
    if not isinstance(x, torch.Tensor) or not isinstance(log_decay, torch.Tensor):
        raise TypeError(f"{what} and log_decay must be tensors")
    code, g_code = _lib.DTYPE_CODES.get(x.dtype), _lib.DTYPE_CODES.get(log_decay.dtype)
    if code is None:
        raise TypeError(f"{what} must be fp32, bf16 or fp16, got {x.dtype}")
    if g_code != code and g_code != _lib.DTYPE_F32:
        raise TypeError(f"log_decay must be {x.dtype} or fp32, got {log_decay.dtype}")
    index = x.get_device()
    if index < 0 or log_decay.get_device() != index:
        raise ValueError(f"{what} and log_decay must be CUDA tensors on one device")
    index = _lib.device_index(x, what)
    lead = 2 if cu_seqlens is None else 1
    shape = tuple(x.shape)
    dims = len(shape) - lead
    if dims == 2:
        heads, d = shape[-2], shape[-1]
    elif dims == 1:
        heads, d = 1, shape[-1]
    else:
        raise ValueError(f"{what} must be [B, T, C] or [B, T, H, d] (packed: [N, C] or [N, H, d])")
    shared = dims == 2 and log_decay.dim() == lead + 1
    if log_decay.shape != (shape[:-1] if shared else shape):
        raise ValueError(f"log_decay must have {what}'s shape, or one value per head of [.., H, d]")
    if shared and d not in (32, 64, 128):
        raise ValueError("a decay per head needs a head dim of 32, 64 or 128 (expand it per channel for others)")
    if cu_seqlens is None:
        seqs, rows = shape[0], shape[1]
    else:
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.get_device() != index:
            raise ValueError("cu_seqlens must be int32 [sequences + 1] on the device of the rows")
        if cu_seqlens.numel() < 1 or not cu_seqlens.is_contiguous():
            raise ValueError("cu_seqlens must be contiguous and hold at least one offset")
        seqs, rows = cu_seqlens.numel() - 1, shape[0]
    state_shape = (seqs, *shape[lead:])
    if state is not None:
        _check_state(state, index, state_shape, "state")
    return index, code, g_code, lead, seqs, rows, heads, d, shared, state_shape


def _check_state(state, index, shape, name):
    if state.dtype != torch.float32 or state.get_device() != index:
        raise TypeError(f"{name} must be fp32 on the device of the rows")
    if state.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(state.shape)}")


def _dense(shape, lead, channels):
    """(batch stride, row stride) of a contiguous tensor, as _rows gives them."""
    if lead == 1:
        return 0, channels if shape[0] > 1 else 0
    return channels * shape[1] if shape[0] > 1 else 0, channels if shape[1] > 1 else 0


def _rows(t, lead, channels):
    """(t with each row's channels contiguous, copied if they are not; batch stride; row
    stride).  A stride that no index multiplies counts as 0."""
    shape = t.shape
    if t.is_contiguous():
        return t, *_dense(shape, lead, channels)
    need = 1
    for n, s in zip(reversed(shape[lead:]), reversed(t.stride()[lead:])):
        if n != 1 and s != need:
            t = t.contiguous()
            break
        need *= n
    stride = t.stride()
    row = stride[lead - 1] if shape[lead - 1] > 1 else 0
    return t, (stride[0] if shape[0] > 1 else 0) if lead == 2 else 0, row


def _aligned(t, batch, row, lead, d):
    """_rows's result with rows that start at whole vectors of d / 32 values, copied if they do not
    (a lane of the shared-decay kernels owns that many)."""
    vec = d // 32
    if vec > 1 and (batch % vec or row % vec or t.data_ptr() % (vec * t.element_size())):
        return _rows(t.clone(memory_format=torch.contiguous_format), lead, t.shape[lead:].numel())
    return t, batch, row


def _span(t):
    """(first address, the one behind the last) of t's values."""
    start = t.data_ptr()
    if t.is_contiguous():
        return start, start + t.nbytes
    return start, start + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _meets(a, b):
    """Whether the address ranges of a and b meet."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1 and a.numel() > 0 and b.numel() > 0


def _same(a, b):
    return a.data_ptr() == b.data_ptr() and a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()


def _beside(a, b, lead):
    """Whether a and b, rows of one buffer at the same strides, are different parts of each of its periods
    (columns of the same rows, every other row, every other batch): no address in both."""
    if a.element_size() != b.element_size() or a.shape[:lead] != b.shape[:lead]:
        return False
    dims = sorted((q, n) for n, p, q in zip(a.shape[:lead], a.stride(), b.stride()) if n > 1 and p == q)
    if len(dims) != sum(n > 1 for n in a.shape[:lead]):
        return False
    off = (b.data_ptr() - a.data_ptr()) // a.element_size()
    inner = 0                                         # what the smaller strides span
    for i, (pitch, n) in enumerate(dims):
        if pitch > 0 and all(p % pitch == 0 for p, _ in dims[i:]):
            first = off % pitch
            if first >= inner + a.shape[lead:].numel() and first + inner + b.shape[lead:].numel() <= pitch:
                return True
        inner += (n - 1) * pitch
    return False


def _check_memory(x, log_decay, state, out, out_state, lead):
    """Refuses outputs whose memory a row or state still to be read, or another output, shares: the
    order in which rows are read and written is not that of the recurrence."""
    step = lead == 2 and x.shape[1] == 1              # each value is read and written by one thread
    if out is not None:
        for n, s in zip(out.shape[:lead], out.stride()):
            if n > 1 and s < out.shape[lead:].numel():
                raise ValueError("out's rows must not overlap")
        for t, name in ((x, "x"), (log_decay, "log_decay")):
            if _meets(out, t) and not _same(out, t) and not _beside(out, t, lead):
                raise ValueError(f"out and {name} must be the same rows or share no memory")
        for t, name in ((state, "state"), (out_state, "out_state")):
            if t is not None and _meets(out, t) and not (step and out.data_ptr() == t.data_ptr() and
                                                         out.dtype == t.dtype and out.is_contiguous()):
                raise ValueError(f"out and {name} must not share memory")
    if out_state is not None:
        if state is not None and out_state is not state and _meets(out_state, state) and not _same(out_state, state):
            raise ValueError("out_state and state must be the same memory or share none")
        for t, name in ((x, "x"), (log_decay, "log_decay")):
            if _meets(out_state, t) and not (step and out_state.data_ptr() == t.data_ptr() and t.dtype == torch.float32 and
                                             t.numel() == out_state.numel() and t.is_contiguous()):
                raise ValueError(f"out_state and {name} must not share memory")


def _forward(x, log_decay, state, cu_seqlens, reverse, out, out_state):
    _lib.refuse_tangents("gated_scan", x, log_decay, state, out, out_state)
    index, code, g_code, lead, seqs, rows, heads, d, shared, shape = _layout(x, log_decay, state, cu_seqlens, "x")
    device, channels = x.device, heads * d
    given = [t for t in (out, out_state) if t is not None]
    own_state = out_state
    if out is None:
        y = torch.empty(x.shape, dtype=x.dtype, device=device)
        y_batch, y_row = _dense((seqs, rows) if lead == 2 else (rows,), lead, channels)
    else:
        y = out
        if out.shape != x.shape or out.dtype != x.dtype or out.get_device() != index:
            raise ValueError("out must match x in shape, dtype and device")
        whole, y_batch, y_row = _rows(out, lead, channels)
        if whole is not out:
            raise ValueError("out's channels must be contiguous")
    if out_state is None:
        out_state = torch.empty(shape, dtype=torch.float32, device=device)
    else:
        _check_state(out_state, index, shape, "out_state")
        if not out_state.is_contiguous():
            raise ValueError("out_state must be contiguous")
    if channels == 0:
        return y, out_state
    if seqs == 0:
        return (y.zero_() if out is None else y), out_state
    x, x_batch, x_row = _rows(x, lead, channels)
    if shared:
        x, x_batch, x_row = _aligned(x, x_batch, x_row, lead, d)
    log_decay, g_batch, g_row = _rows(log_decay, lead, heads if shared else channels)
    if state is not None and not state.is_contiguous():
        state = state.contiguous()
    if given:
        _check_memory(x, log_decay, state, out, own_state, lead)
    _lib.call_on(index, "vdn_gated_scan", x.data_ptr(), code, x_batch, x_row, log_decay.data_ptr(), g_code, g_batch,
                 g_row, shared, None if state is None else state.data_ptr(),
                 None if cu_seqlens is None else cu_seqlens.data_ptr(), seqs, rows, heads, d, reverse, y.data_ptr(),
                 y_batch, y_row, out is None, out_state.data_ptr(), _lib.status_word(index))
    if given:                                        # written past autograd's sight: graphs that saved them must fail
        torch.autograd.graph.increment_version(given)
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
        _lib.refuse_captured_autograd("gated_scan", ctx.saved_tensors[0])
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
    sequences lie end to end: x [N, C] or [N, H, d]; rows in front of the first offset and
    behind the last come back zero, and stay as they were in a caller's `out`.  state / out_state fp32 [B or S, C] or
    [.., H, d]; out_state may be `state` and out may be x or log_decay (updated in place); other shared
    memory is refused.  reverse runs each sequence from
    its last row to its first.  Strided rows and expanded log_decay are read in place as
    long as a row's channels are contiguous.  A state that overflows fp32 comes out as inf or NaN.
    exp(log_decay) counts as 0 below -87.7 and as inf above 88.37.  Decays may grow (log_decay above 0), but up to
    256 tokens in a row are folded into one factor: where a product of successive decays among them leaves
    fp32's range, the state carried in counts as 0 (below the range) or gives inf or NaN (above), even if the
    states themselves would have stayed inside.
    """
    if torch.is_grad_enabled() and _lib.records(x, log_decay, state, out, out_state):
        if out is not None or out_state is not None:
            raise ValueError("out and out_state cannot be given where gradients are recorded")
        _lib.refuse_captured_autograd("gated_scan", x)
        return _GatedScan.apply(x, log_decay, state, cu_seqlens, bool(reverse))
    return _forward(x, log_decay, state, cu_seqlens, bool(reverse), out, out_state)


def gated_scan_backward(grad_y, log_decay, y, *, state=None, grad_state=None, cu_seqlens=None, reverse=False):
    """(grad of x, of log_decay, of state) from the forward's output y and its arguments.

    grad_state is the gradient of the last state, if any; the gradient of the first state
    comes back as fp32 also when `state` was None.  Rows outside the packed sequences
    have zero gradients.  Records nothing for autograd."""
    return _backward(grad_y, log_decay, y, state, grad_state, cu_seqlens, bool(reverse))


def _backward(grad_y, log_decay, y, state, grad_state, cu_seqlens, reverse):
    _lib.refuse_tangents("gated_scan_backward", grad_y, log_decay, y, state, grad_state)
    index, code, g_code, lead, seqs, rows, heads, d, shared, shape = _layout(y, log_decay, state, cu_seqlens, "y")
    if grad_y.shape != y.shape or grad_y.dtype != y.dtype or grad_y.get_device() != index:
        raise ValueError("grad_y must match y in shape, dtype and device")
    if grad_state is not None:
        _check_state(grad_state, index, shape, "grad_state")
        grad_state = grad_state.contiguous()
    device, channels = y.device, heads * d
    dx = torch.empty(y.shape, dtype=y.dtype, device=device)
    dg = torch.empty(log_decay.shape, dtype=log_decay.dtype, device=device)
    ds = torch.empty(shape, dtype=torch.float32, device=device)
    if channels == 0 or seqs == 0:
        return dx.zero_(), dg.zero_(), ds
    decays = heads if shared else channels
    grad_y, dy_batch, dy_row = _rows(grad_y, lead, channels)
    log_decay, g_batch, g_row = _rows(log_decay, lead, decays)
    y, y_batch, y_row = _rows(y, lead, channels)
    if shared:
        grad_y, dy_batch, dy_row = _aligned(grad_y, dy_batch, dy_row, lead, d)
        y, y_batch, y_row = _aligned(y, y_batch, y_row, lead, d)
    lead_shape = (seqs, rows) if lead == 2 else (rows,)
    dx_batch, dx_row = _dense(lead_shape, lead, channels)
    dg_batch, dg_row = _dense(lead_shape, lead, decays)
    if state is not None and not state.is_contiguous():
        state = state.contiguous()
    _lib.call_on(index, "vdn_gated_scan_backward", grad_y.data_ptr(), code, dy_batch, dy_row, log_decay.data_ptr(),
                 g_code, g_batch, g_row, shared, y.data_ptr(), y_batch, y_row, None if state is None else state.data_ptr(),
                 None if grad_state is None else grad_state.data_ptr(),
                 None if cu_seqlens is None else cu_seqlens.data_ptr(), seqs, rows, heads, d, reverse, dx.data_ptr(),
                 dx_batch, dx_row, dg.data_ptr(), dg_batch, dg_row, True, ds.data_ptr(), _lib.status_word(index))
    return dx, dg, ds
