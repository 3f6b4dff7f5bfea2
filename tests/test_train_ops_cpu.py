"""CPU: the differentiable operators' argument checks (Python and C ABI), workspace sizes, and the
call path's handling of devices and captures."""
import ctypes as C
import types

import pytest
import torch

from vdn_b200 import _lib
from vdn_b200.layer_norm import layer_norm, layer_norm_backward
from vdn_b200.linear_act import linear_act, linear_act_backward
from vdn_b200.recurrence import gated_scan, gated_scan_backward

BF, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F32
P = 1 << 20                      # an aligned address that no call here dereferences


def _fails(rc, code, text):
    assert rc == code, (rc, _lib.load().vdn_last_error())
    assert text in _lib.load().vdn_last_error().decode()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        gated_scan(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        gated_scan_backward(x, x, x)
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm_backward(x, x, None, torch.zeros(6), torch.zeros(6))
    with pytest.raises(ValueError, match="CUDA"):
        linear_act(x, x[0])
    with pytest.raises(ValueError, match="CUDA"):
        linear_act_backward(x, x, torch.zeros(64, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA"):                     # also where gradients would be recorded
        layer_norm(x.clone().requires_grad_())


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.float8_e4m3fn])
def test_types_are_refused(dtype):
    x = torch.zeros(2, 3, 64).to(dtype)
    for call in (lambda: gated_scan(x, x), lambda: layer_norm(x), lambda: linear_act(x, x[0])):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: gated_scan(None, x), lambda: layer_norm(None), lambda: linear_act(None, x)):
        with pytest.raises(TypeError):
            call()


def _scan(dtype=BF, g_dtype=BF, shared=0, seqs=1, rows=4, heads=2, d=32, row=64, x=P):
    return _lib.load().vdn_gated_scan(x, dtype, row * rows, row, P, g_dtype, row * rows, row, shared, None, None, seqs,
                                      rows, heads, d, 0, P, row * rows, row, 0, None, None, None)


def test_scan_abi_checks():
    _fails(_scan(dtype=7), _lib.VDN_ERR_TYPE, "dtype")
    _fails(_scan(g_dtype=_lib.DTYPE_F16), _lib.VDN_ERR_TYPE, "log_decay")
    _fails(_scan(shared=1, d=48), _lib.VDN_ERR_VALUE, "32, 64 or 128")
    _fails(_scan(row=1 << 26), _lib.VDN_ERR_VALUE, "2^26")
    _fails(_scan(rows=-1), _lib.VDN_ERR_VALUE, "extents")
    _fails(_scan(rows=1 << 30), _lib.VDN_ERR_VALUE, "large")
    _fails(_scan(x=None), _lib.VDN_ERR_VALUE, "null")
    assert _scan(seqs=0) == _lib.VDN_OK and _scan(rows=0) == _lib.VDN_OK
    back = _lib.load().vdn_gated_scan_backward
    args = [P, BF, 64, 64, P, BF, 64, 64, 0, P, 64, 64, None, None, None, 1, 1, 1, 64, 0, P, 64, 64, None, 64, 64, 0,
            None, None, None]
    _fails(back(*args), _lib.VDN_ERR_VALUE, "null")


def test_layer_norm_abi_checks():
    lib = _lib.load()
    _fails(lib.vdn_layer_norm(P, 9, 4, 64, 64, None, None, F32, 1e-5, P, 64, None, None, None), _lib.VDN_ERR_TYPE, "dtype")
    _fails(lib.vdn_layer_norm(P, F32, 4, 64, 64, None, None, BF, 1e-5, P, 64, None, None, None), _lib.VDN_ERR_TYPE, "weight")
    _fails(lib.vdn_layer_norm(P, BF, 4, 0, 64, None, None, BF, 1e-5, P, 64, None, None, None), _lib.VDN_ERR_VALUE, "extents")
    _fails(lib.vdn_layer_norm(P, BF, 4, 64, 64, None, None, BF, 1e-5, P, 32, None, None, None), _lib.VDN_ERR_VALUE, "stride")
    assert lib.vdn_layer_norm(None, BF, 0, 64, 64, None, None, BF, 1e-5, None, 64, None, None, None) == _lib.VDN_OK
    need = lib.vdn_layer_norm_backward_workspace_size
    assert need(0, 64) == 0 and need(4, 0) == 0
    assert need(4, 64) == 4 * 2 * 4 * 64                              # a line per row, no more
    for width in (64, 1000, 1280, 3584, 5120, 16384, 40000):          # bounded whatever the rows
        assert need(1 << 20, width) == need(1 << 24, width) <= 2960 * 2 * 4 * width
    rc = lib.vdn_layer_norm_backward(P, BF, 4, 64, 64, P, 64, None, BF, P, P, P, 64, None, None, P, need(4, 64) - 1, None,
                                     None)
    _fails(rc, _lib.VDN_ERR_VALUE, "workspace")


def test_linear_abi_checks():
    lib = _lib.load()

    def linear(dtype=BF, act=0, x=P, ldx=64, k=64, ws=0, y=P + (1 << 16), residual=None):
        return lib.vdn_linear_act(x, ldx, P, 64, None, residual, 64, dtype, act, 4, 64, k, y, 64, None, 0, None, ws, None,
                                  None)
    _fails(linear(dtype=F32), _lib.VDN_ERR_TYPE, "bf16 or fp16")
    _fails(linear(act=_lib.ACT_SWIGLU), _lib.VDN_ERR_VALUE, "activation")
    _fails(linear(x=None), _lib.VDN_ERR_VALUE, "null")
    _fails(linear(residual=P + (1 << 16)), _lib.VDN_ERR_VALUE, "overlap")
    _fails(linear(x=P + 2), _lib.VDN_ERR_VALUE, "workspace")          # not 16-byte aligned: copied first
    _fails(linear(ldx=65), _lib.VDN_ERR_VALUE, "workspace")
    size = lib.vdn_linear_workspace_size
    assert size(P, 64, P, 64, 4, 64, 64) == 0
    assert size(P + 2, 64, P, 64, 4, 64, 64) == 512                   # 4 rows of 64 values
    assert size(P, 61, P, 61, 3, 5, 61) == 512 + 768                  # rows padded to 64 values, 256-byte pieces
    rc = lib.vdn_linear_act_backward(P, 64, None, 0, P, 64, P, 64, BF, _lib.ACT_SILU, 4, 64, 64, P, 64, P, 64, None, None,
                                     0, None, None)
    _fails(rc, _lib.VDN_ERR_VALUE, "null")
    rc = lib.vdn_linear_act_backward(P, 64, P, 64, P, 64, P, 64, BF, _lib.ACT_SILU, 4, 64, 64, P, 64, P, 64, None, None,
                                     0, None, None)
    _fails(rc, _lib.VDN_ERR_VALUE, "workspace")


def test_calls_run_on_the_tensors_device(monkeypatch):
    """call_on makes the tensors' device current for the call and passes its current stream."""
    seen, current = [], [0]

    class Device:
        def __init__(self, d):
            self.d = d

        def __enter__(self):
            self.before, current[0] = current[0], self.d

        def __exit__(self, *exc):
            current[0] = self.before
    monkeypatch.setattr(_lib, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(_lib, "_raw_stream", lambda index: 1000 + index)
    monkeypatch.setitem(_lib._FUNCTIONS, "vdn_fake", lambda *a: seen.append((current[0], a)) or 0)
    _lib.call_on(0, "vdn_fake", 5)
    _lib.call_on(3, "vdn_fake", 6)
    assert seen == [(0, (5, 1000)), (3, (6, 1003))] and current == [0]
    monkeypatch.setitem(_lib._FUNCTIONS, "vdn_fake", lambda *a: _lib.VDN_ERR_VALUE)
    with pytest.raises(ValueError):
        _lib.call_on(3, "vdn_fake")
    assert current == [0]


def test_no_status_word_is_made_inside_a_capture(monkeypatch):
    from vdn_b200 import mxfp8_linear as ml
    monkeypatch.setattr(ml, "_STATUS", {})
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert ml.status_address(torch.device("cuda", 0)) is None and not ml._STATUS
    with pytest.raises(RuntimeError, match="capture"):
        _lib.refuse_captured_autograd("layer_norm", types.SimpleNamespace(device=torch.device("cuda", 0)))
    word = torch.zeros(1, dtype=torch.int32)
    ml._STATUS[0] = word
    assert ml.status_address(torch.device("cuda", 0)) == word.data_ptr()
    assert C.c_int32.from_address(word.data_ptr()).value == 0
