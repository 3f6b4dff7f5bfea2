"""GPU: the scan's error against 64 bits, held to what its arithmetic gives.

With u = 2^-24.  The decay is a pair hi + lo within 2.5e-8 = 0.42u of exp(g), relative.  A step rounds twice
(x + lo h, then hi h + that: u/2 each of values at most M_t, the recurrence on absolute values).  A carry reaches token l
through the product of the hi parts (0.42u, u/2 for hi and u/2 for the product a token).  Joining a warp's run of
16 or 32 tokens and a CTA's run of up to 256 rounds some six times more, and the run's factor errs by at most u a
token, whether it comes from the sum of its decays (at most 2) or from their product.  Together below 3u M_t a token."""
import pytest
import torch

import test_recurrence_gpu as base
from test_recurrence_gpu import TYPES, U, _case, _run

pytestmark = pytest.mark.gpu


@pytest.fixture
def tight(monkeypatch):
    """test_recurrence_gpu's reference with 3u a token in place of 8u."""
    wide = base._reference

    def reference(*args):
        res = wide(*args)
        return {k: v * (3 / 8) if k.endswith("_err") else v for k, v in res.items()}
    monkeypatch.setattr(base, "_reference", reference)


@pytest.mark.parametrize("tokens,heads,d,shared", [(700, 2, 64, False), (700, 2, 64, True), (2500, 1, 64, False), (2500, 1, 128, True),
                                                   (600, 1, 61, False), (2100, 1, 32, True)])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("sharp", [False, True])
def test_three_units_a_token(cuda, tight, tokens, heads, d, shared, reverse, sharp):
    gen, x, g = _case(tokens + d, (1, tokens), heads, d, torch.float32, torch.float32, shared, sharp=sharp)
    _run(cuda, x, g, None, reverse, True, gen)


@pytest.mark.parametrize("dtype,g_dtype", TYPES)
def test_three_units_a_token_packed(cuda, tight, dtype, g_dtype):
    gen, x, g = _case(77, (1500,), 2, 64, dtype, g_dtype, False)
    _run(cuda, x, g, [0, 3, 900, 900, 1499], False, True, gen)


def _rounded_far(count):
    """log decays near -2^-10 whose exponentials lie almost half a unit from fp32's: hi alone errs by that
    at every token, in one direction."""
    g = -torch.arange(8192, 8192 + 60000, dtype=torch.float64).mul(2.0 ** -23).float()
    a = g.double().exp()
    off = (a.float().double() - a) / 2.0 ** -24
    g, off = g[off > 0.49], off[off > 0.49]
    assert len(g) >= count
    return g[:count], off[:count]


@pytest.mark.parametrize("tokens,span,channels", [(16, 16, 4096), (2048, 32, 2048)])       # one run of 16, the last run of 32
@pytest.mark.parametrize("shared", [False, True])
def test_low_parts_of_the_decays_count(cuda, tokens, span, channels, shared):
    """An impulse decays over one run.  Its mean relative error over the channels, whose mantissas differ, is
    the decays' own: roundings of either sign average out (u/2 sqrt(span / channels), six times that allowed), and the
    pair errs by 0.42u of 1 - a only.  Without the low parts the error would be 0.49u a token."""
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    gen = torch.Generator().manual_seed(9)
    limit = 6 * 0.5 * (span / channels) ** 0.5 + 0.01 * span
    assert limit < 0.2 * 0.49 * (span - 1)
    decays, _ = _rounded_far(3)
    for value in decays:
        heads = channels // 64
        g = torch.full((1, tokens, heads) if shared else (1, tokens, heads, 64), float(value))
        impulse = torch.rand(heads, 64, generator=gen) + 1
        x = torch.zeros(1, tokens, heads, 64)
        x[0, tokens - span] = impulse
        y, last = gated_scan(x.to(cuda), g.to(cuda))
        want = impulse.double() * (value.double() * (span - 1)).exp()
        off = ((last[0].double().cpu() - want) / want).mean() / U
        assert abs(float(off)) < limit, float(off)
        dy = torch.zeros_like(x)                           # backwards the last run walked holds the first tokens
        dy[0, span - 1] = impulse
        _, _, ds = gated_scan_backward(dy.to(cuda), g.to(cuda), y)
        want = impulse.double() * (value.double() * span).exp()
        off = ((ds[0].double().cpu() - want) / want).mean() / U
        assert abs(float(off)) < limit, float(off)


def test_constant_slow_decay_in_joins_of_128(cuda):
    """test_constant_slow_decay_keeps_its_memory with the joins that this shape takes: runs of 32 tokens, four warps
    a CTA, so 16400 / 128 = 128 joins are remembered.  Each rounds the run's factor (u/2 and 0.42u of its distance from 1)
    and the state (u/2).  A CTA's own fold reaches over 128 tokens by products of hi parts: u a token, half
    of them on average, and u/2 a step of a warp's own run.  (129 + 64 + 8) u = 1.2e-5."""
    from vdn_b200.recurrence import gated_scan
    n = 60000
    for value in (-1.0 / 16400, -1.0 / 16000, -1.0 / 15777):
        g = torch.full((1, n, 64), value)
        _, last = gated_scan(torch.ones(1, n, 64, device=cuda), g.to(cuda))
        a = g[0, 0, 0].double().exp()
        want = (1 - a ** n) / (1 - a)
        assert float((last.double().cpu() - want).abs().max() / want) < 201 * U
