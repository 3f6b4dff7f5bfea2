"""GPU: the state carried through strong decays or growth keeps its relative accuracy.

Without inputs the last state is the first one times the product of n decays.  Each decay is within 0.42u of
exp(g), and each step (or each factor of a run's product) rounds at most twice: 2u a token covers both, u = 2^-24, and
six more roundings join runs, warps and CTAs.  A factor taken from a rounded sum of decays would err by half a unit
of the sum, 32u at -62, however few the tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("tokens", [2, 3, 7, 40, 150, 1100])
@pytest.mark.parametrize("shared,d", [(False, 64), (False, 33), (True, 64), (True, 128)])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_products_of_decays(cuda, tokens, shared, d, sign):
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    gen = torch.Generator().manual_seed(tokens)
    heads = 4
    shape = (1, tokens, heads) if shared else (1, tokens, heads, d)
    g = torch.rand(shape, generator=gen)
    g = g / g.sum(1, keepdim=True) * (20 + 55 * torch.rand(shape[:1] + shape[2:], generator=gen))[:, None] * sign
    state = torch.randn(1, heads, d, generator=gen)
    x = torch.zeros(1, tokens, heads, d)
    total = g.double().sum(1)
    want = state.double() * (total[..., None] if shared else total).exp()
    err = (2 * tokens + 6) * U * want.abs()
    y, last = gated_scan(x.to(cuda), g.to(cuda), state.to(cuda))
    assert bool(((last.double().cpu() - want).abs() <= err).all()), float(((last.double().cpu() - want) / want).abs().max() / U)
    _, _, ds = gated_scan_backward(torch.zeros_like(y), g.to(cuda), y, state=state.to(cuda), grad_state=state.to(cuda))
    assert bool(((ds.double().cpu() - want).abs() <= err).all()), float(((ds.double().cpu() - want) / want).abs().max() / U)


def test_steps_and_one_call_agree(cuda):
    """Tokens served one by one and in one call end in the same state, strong decays or not."""
    from vdn_b200.recurrence import gated_scan
    gen = torch.Generator().manual_seed(3)
    for scale in (0.01, 1.0, 12.0):
        g = (-scale * torch.rand(2, 6, 128, generator=gen)).to(cuda)
        state = torch.randn(2, 128, generator=gen).to(cuda)
        x = torch.zeros_like(g)
        _, want = gated_scan(x, g, state)
        for t in range(6):
            _, state = gated_scan(x[:, t:t + 1], g[:, t:t + 1], state)
        assert bool(((state - want).abs() <= 2 * (2 * 6 + 6) * U * want.abs()).all())
