"""The per-token operators and what autograd asks of them beside reverse-mode gradients."""
import pytest
import torch
from torch.autograd import forward_ad

from vdn_b200.layer_norm import layer_norm, layer_norm_backward
from vdn_b200.linear_act import linear_act, linear_act_backward
from vdn_b200.recurrence import gated_scan, gated_scan_backward


def _tangents(dev):
    x = torch.randn(2, 3, 64, generator=torch.Generator().manual_seed(0)).bfloat16().to(dev)
    w = torch.zeros(64, 64, dtype=torch.bfloat16, device=dev)
    state, rows = torch.zeros(2, 64, device=dev), torch.ones(6, device=dev)
    calls = [
        (x, lambda t: gated_scan(t, x)), (x, lambda t: gated_scan(x, t)), (state, lambda t: gated_scan(x, x, t)),
        (x, lambda t: gated_scan(x, x, out=t)), (state, lambda t: gated_scan(x, x, out_state=t)),
        (x, lambda t: gated_scan_backward(t, x, x)), (x, lambda t: gated_scan_backward(x, t, x)),
        (state, lambda t: gated_scan_backward(x, x, x, grad_state=t)),
        (x, layer_norm), (x[0, 0], lambda t: layer_norm(x, t)), (x[0, 0], lambda t: layer_norm(x, None, t)),
        (x, lambda t: layer_norm_backward(t, x, None, rows, rows)),
        (rows, lambda t: layer_norm_backward(x, x, None, rows, t)),
        (x, lambda t: linear_act(t, w)), (w, lambda t: linear_act(x, t)), (w[0], lambda t: linear_act(x, w, t)),
        (x, lambda t: linear_act(x, w, residual=t)),
        (x, lambda t: linear_act_backward(t, x, w)), (w, lambda t: linear_act_backward(x, x, t)),
    ]
    with forward_ad.dual_level():
        for t, call in calls:
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward-mode"):
                    call(forward_ad.make_dual(t, torch.ones_like(t)))
    return x


def test_tangents_are_refused_on_the_cpu():
    _tangents("cpu")


@pytest.mark.gpu
def test_tangents_are_refused(cuda):
    x = _tangents(cuda)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):       # where gradients are recorded as well
        layer_norm(forward_ad.make_dual(x.clone().requires_grad_(), torch.ones_like(x)))
    with forward_ad.dual_level():                          # a level alone changes nothing
        assert torch.equal(layer_norm(x), layer_norm(x.clone()))
        gated_scan(x, x, out=torch.empty_like(x))
