"""GPU: what a call writes into the caller's tensors (`out`, `out_state`) is seen by autograd."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _args(cuda, tokens=5):
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(2, tokens, 2, 64, generator=gen).to(cuda)
    g = -torch.rand(2, tokens, 2, 64, generator=gen).to(cuda)
    return x, g, torch.randn(2, 2, 64, generator=gen).to(cuda)


@pytest.mark.parametrize("tokens", [1, 5])
def test_saved_state_written_over_is_an_error(cuda, tokens):
    """The gradient of log_decay needs the first state: a later step into its memory must not pass unnoticed."""
    from vdn_b200.recurrence import gated_scan
    x, g, state = _args(cuda, tokens)
    leaf = g.clone().requires_grad_()
    y, _ = gated_scan(x, leaf, state)
    with torch.no_grad():
        gated_scan(x[:, :1], g[:, :1], state, out_state=state)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    y, _ = gated_scan(x, leaf, state.clone())              # a copy is left alone
    with torch.no_grad():
        gated_scan(x[:, :1], g[:, :1], state, out_state=state)
    y.sum().backward()
    assert bool(torch.isfinite(leaf.grad).all())


def test_saved_decay_or_output_written_over_is_an_error(cuda):
    from vdn_b200.recurrence import gated_scan
    x, g, state = _args(cuda)
    for pick in ("decay", "output"):
        decay = g.clone()
        y, _ = gated_scan(x.clone().requires_grad_(), decay, state)
        with torch.no_grad():
            gated_scan(x, g, out=decay if pick == "decay" else y.detach())
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()


def test_outputs_that_need_gradients_are_refused(cuda):
    from vdn_b200.recurrence import gated_scan
    x, g, state = _args(cuda)
    with pytest.raises(ValueError, match="recorded"):
        gated_scan(x, g, state, out=torch.empty_like(x).requires_grad_())
    with pytest.raises(ValueError, match="recorded"):
        gated_scan(x, g, state, out_state=state.clone().requires_grad_())
    with torch.no_grad():
        gated_scan(x, g, state, out=torch.empty_like(x).requires_grad_())
    with torch.inference_mode():                           # tensors without a version counter
        out = torch.empty_like(x)
        y, _ = gated_scan(x, g, state, out=out)
    assert y is out
