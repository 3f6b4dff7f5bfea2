"""CPU: workspaces that the kernels' vector stores could not take are refused before any launch.
The addresses are never dereferenced: every call here ends in the argument checks."""
import pytest

from vdn_b200 import _lib

BF, SILU, NONE = _lib.DTYPE_BF16, _lib.ACT_SILU, _lib.ACT_NONE
P, WS = 1 << 20, 1 << 24


def _refused(rc):
    assert rc == _lib.VDN_ERR_VALUE and "aligned" in _lib.load().vdn_last_error().decode(), (rc, _lib.load().vdn_last_error())


@pytest.mark.parametrize("off", [2, 4, 8])
def test_linear_workspace(off):
    lib = _lib.load()
    _refused(lib.vdn_linear_act(P + 2, 64, P, 64, None, None, 0, BF, NONE, 4, 64, 64, P + 4096, 64, None, 0, WS + off, 1 << 20,
                                None, None))
    for dy, act in ((P + 2, NONE), (P, SILU)):            # dy copied; dz written
        _refused(lib.vdn_linear_act_backward(dy, 64, P, 64, P, 64, P, 64, BF, act, 4, 64, 64, P + 4096, 64, None, 0, None,
                                             WS + off, 1 << 20, None, None))


def test_partial_sums_workspace():
    lib = _lib.load()
    _refused(lib.vdn_linear_act_backward(P, 64, None, 0, P, 64, P, 64, BF, NONE, 4, 64, 64, None, 0, None, 0, P + 4096,
                                         WS + 2, 1 << 20, None, None))
    _refused(lib.vdn_layer_norm_backward(P, BF, 4, 64, 64, P, 64, None, BF, P, P, P + 4096, 64, None, None, WS + 2, 1 << 20,
                                         None, None))
