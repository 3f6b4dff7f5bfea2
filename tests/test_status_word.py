"""A wait that gave up inside a per-token operator's kernel is reported by the operators themselves.

Waits are made to run out on the host (a fake word) or by a fence whose flag nothing sets: it
gives up after its limit and writes the status word it was given, which is the operators' own."""
import ctypes as C
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import vdn_b200
from vdn_b200 import _lib

ROOT = Path(__file__).resolve().parents[1]


def test_a_set_word_raises_once(monkeypatch):
    word = C.c_int32(0)
    monkeypatch.setattr(_lib, "_WORDS", {3: word})
    assert _lib.status_word(3) == C.addressof(word)
    word.value = _lib.VDN_ERR_TIMEOUT
    with pytest.raises(RuntimeError, match="gave up"):
        _lib.status_word(3)
    assert word.value == 0 and _lib.status_word(3) == C.addressof(word)


def test_check_status_waits_and_reports(monkeypatch):
    word, waited = C.c_int32(_lib.VDN_ERR_TIMEOUT), []
    monkeypatch.setattr(_lib, "_WORDS", {1: word})
    monkeypatch.setattr(torch.cuda, "synchronize", waited.append)
    with pytest.raises(RuntimeError, match="cuda:1"):
        vdn_b200.check_status("cuda:1")
    vdn_b200.check_status(torch.device("cuda", 1))
    assert waited == [1, 1]


def test_bad_devices_are_refused():
    at = C.c_void_p()
    for device in (-1, 64):
        assert _lib.load().vdn_status_word(device, C.byref(at)) == _lib.VDN_ERR_VALUE
    assert _lib.load().vdn_status_word(0, None) == _lib.VDN_ERR_VALUE


def _run_out(cuda, address):
    """A two-rank fence on one GPU whose second flag nothing sets; ends after its own limit."""
    mine, peer = (torch.zeros(16, dtype=torch.int64, device=cuda) for _ in range(2))
    flags = (C.c_void_p * 2)(mine.data_ptr(), peer.data_ptr())
    _lib.call("vdn_peer_fence", 2, flags, C.c_void_p(mine.data_ptr()), 0, C.c_void_p(mine.data_ptr() + 64),
              C.c_void_p(address), _lib.stream_of(cuda))
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_the_device_reaches_the_word(cuda):
    from vdn_b200.linear_act import linear_act
    from vdn_b200.mxfp8_linear import check_gemm_status
    from vdn_b200.recurrence import gated_scan
    x = torch.ones(2, 40, 64, device=cuda)
    want = gated_scan(x, -x)
    at = _lib.status_word(0)
    for report in (lambda: gated_scan(x, -x), lambda: linear_act(x.half(), x[0].half()), lambda: vdn_b200.check_status(cuda)):
        _run_out(cuda, at)
        check_gemm_status(cuda)                            # not the MXFP8 GEMMs' business
        with pytest.raises(RuntimeError, match="gave up"):
            report()
        report()
    assert all(torch.equal(a, b) for a, b in zip(gated_scan(x, -x), want)) and _lib.status_word(0) == at


@pytest.mark.gpu
def test_the_first_call_may_be_captured(cuda):
    """The word is made inside the capture without breaking it, and outlives the graph."""
    code = """
import torch
from vdn_b200 import _lib
from vdn_b200.recurrence import gated_scan
x = torch.ones(2, 40, 64, device="cuda")
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    y, last = gated_scan(x, -x)
at = _lib.status_word(0)
del y, last
graph.replay()
torch.cuda.synchronize()
del graph
assert _lib.status_word(0) == at and _lib._WORDS[0].value == 0
print("captured")
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "captured" in run.stdout, run.stderr
