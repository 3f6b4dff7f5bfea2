"""GPU: log_decay = -inf starts a channel anew whatever the other decays of the run are, growth
(log_decay above 0) among them.

Growth and slow decays are dyadic numbers whose sums fp32 holds exactly, so the bounds of
test_recurrence_gpu.py apply as they stand: nothing in them supposes a decay below 1."""
import pytest
import torch

from test_recurrence_gpu import TYPES, _run

pytestmark = pytest.mark.gpu

INF = float("inf")


def _decays(tokens, tail, growth, count, at, g_dtype):
    """-1/1024 everywhere, `count` tokens of `growth` in front of the restart at row `at`."""
    g = torch.full((tokens, *tail), -1.0 / 1024)
    g[at - count:at] = growth
    g[at] = -INF
    return g.to(g_dtype)


@pytest.mark.parametrize("dtype,g_dtype", TYPES)
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("tokens", [200, 2100])          # runs of 16 and of 32 tokens
@pytest.mark.parametrize("reverse", [False, True])
def test_nothing_passes_a_restart(cuda, dtype, g_dtype, shared, tokens, reverse):
    """Without inputs the state behind a restart is 0, exactly, and so is the gradient in front of it."""
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    at = 20                                               # within the first run, joined with those behind it
    g = _decays(tokens, (2,) if shared else (2, 64), 0.75, 12, at, g_dtype)
    g[at + 1:at + 9] = 0.5                                # growth behind it as well
    gen = torch.Generator().manual_seed(7)
    g = (g.flip(0) if reverse else g)[None].to(cuda)
    state, dlast = (torch.randn(1, 2, 64, generator=gen).to(cuda) for _ in range(2))
    x = torch.zeros(1, tokens, 2, 64, dtype=dtype, device=cuda)
    y, last = gated_scan(x, g, state, reverse=reverse)
    dx, dg, ds = gated_scan_backward(x, g, y, state=state, grad_state=dlast, reverse=reverse)
    turn = (lambda t: t[0].flip(0)) if reverse else (lambda t: t[0])
    assert bool((last == 0).all()) and bool((turn(y)[at:] == 0).all()) and bool((turn(y)[:at] != 0).all())
    assert bool((ds == 0).all()) and bool((turn(dx)[:at] == 0).all())
    assert bool((turn(dx)[at:at + 100] != 0).all()) and bool((turn(dg)[:at + 1] == 0).all())


@pytest.mark.parametrize("dtype,g_dtype", [t for t in TYPES if t[0] != torch.float16])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("growth,count", [(1.0, 80), (5.0, 16), (0.25, 100)])
def test_restart_behind_growth(cuda, dtype, g_dtype, shared, growth, count):
    """States that grow up to e^80 stay inside fp32 and bf16; the rows behind the restart are as if they came first."""
    gen = torch.Generator().manual_seed(3)
    tokens, at = 700, 105
    x = torch.randn(1, tokens, 2, 64, generator=gen).to(dtype)
    g = _decays(tokens, (2,) if shared else (2, 64), growth, count, at, g_dtype)[None]
    _run(cuda, x, g, None, False, True, gen)


def test_restart_behind_growth_packed(cuda):
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(900, 2, 64, generator=gen).bfloat16()
    g = torch.cat([_decays(300, (2,), 1.0, 80, 105, torch.float32), _decays(600, (2,), 5.0, 16, 400, torch.float32)])
    _run(cuda, x, g, [0, 300, 900], False, True, gen)
    _run(cuda, x, g.flip(0), [0, 600, 900], True, True, gen)


def test_lowest_values_are_restarts(cuda):
    """Masks of a type's lowest value count as -inf: their sums overflow to it."""
    from vdn_b200.recurrence import gated_scan
    gen = torch.Generator().manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = torch.randn(2, 300, 64, generator=gen).to(dtype).to(cuda)
        g = torch.full((2, 300, 64), 0.0625).to(dtype)
        g[:, 30:34] = -INF
        low = g.clone()
        low[:, 30:34] = torch.finfo(dtype).min
        want, got = gated_scan(x, g.to(cuda)), gated_scan(x, low.to(cuda))
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert bool(torch.isfinite(want[1]).all())
