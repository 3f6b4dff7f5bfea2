"""GPU: the linear layer's activations and their slopes at values where a formula can go wrong."""
import pytest
import torch

from test_linear_act_gpu import U, _act, _half, _tiny

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["none", "gelu_tanh", "gelu_erf", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,n", [(40, 48), (40, 45), (300, 2056), (300, 2051)])      # vectors and single values
def test_a_nan_stays_in_its_feature(cuda, act, dtype, rows, n):
    """One NaN in pre (the neighbours of its 16-byte vector included): only its feature's dw and bias gradient
    and its row's dx are NaN; without an activation pre is not read."""
    from vdn_b200.linear_act import linear_act, linear_act_backward
    gen = torch.Generator().manual_seed(n)
    x, w = torch.randn(rows, 64, generator=gen).to(dtype).to(cuda), torch.randn(n, 64, generator=gen).to(dtype).to(cuda)
    dy = torch.randn(rows, n, generator=gen).to(dtype).to(cuda)
    _, pre = linear_act(x, w, act=act, return_pre=True)
    want = linear_act_backward(dy, x, w, pre, act=act)
    pre = pre.clone()
    for row, col in ((3, 0), (7, 9), (rows - 1, n - 2)):
        pre[row, col] = float("nan")
    dx, dw, db = linear_act_backward(dy, x, w, pre, act=act)
    rows_off, cols_off = torch.ones(rows, dtype=torch.bool, device=cuda), torch.ones(n, dtype=torch.bool, device=cuda)
    if act != "none":
        rows_off[[3, 7, rows - 1]] = False
        cols_off[[0, 9, n - 2]] = False
        assert bool(torch.isnan(dx[~rows_off]).all() and torch.isnan(dw[~cols_off]).all() and torch.isnan(db[~cols_off]).all())
    assert torch.equal(dx[rows_off], want[0][rows_off]) and torch.equal(dw[cols_off], want[1][cols_off])
    assert torch.equal(db[cols_off], want[2][cols_off])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,n", [(257, 24), (2570, 1032), (257, 21)])      # narrow and pair kernels, single values
def test_exact_gelu_in_its_lower_tail(cuda, dtype, rows, n):
    """z exact (a one-hot product), from -12 to 12: value and slope hold a relative bound down to the type's
    smallest steps.  erfc and exp err by 8u at most, and by z^2 times their argument's rounding (2u each);
    the slope adds cdf and z pdf, whose magnitudes bound it."""
    from vdn_b200.linear_act import linear_act, linear_act_backward
    h, tiny = _half(dtype), _tiny(dtype)
    z = (torch.arange(rows) % 257 - 128.0).div(128 / 12).to(dtype)
    x = torch.zeros(rows, 64, dtype=dtype)
    x[:, 0] = z
    w = torch.zeros(n, 64, dtype=dtype)
    w[:, 0] = 1
    y, pre = linear_act(x.to(cuda), w.to(cuda), act="gelu_erf", return_pre=True)
    zd = z.double()[:, None]
    value, slope = _act(zd, "gelu_erf")
    err = (4 * zd.square() + 20) * U
    assert bool((pre.cpu() == z[:, None]).all())
    bad = (y.double().cpu() - value).abs() - (value.abs() * (h + err * (1 + h)) + tiny)
    assert bool((bad <= 0).all()), (z[bad.amax(1) > 0], y[:, 0].cpu()[bad.amax(1) > 0])
    dy = torch.zeros(rows, n, dtype=dtype)
    dy[:, 1] = 1                                           # dx[:, 0] = the slope, rounded as dz and again
    dx, _, db = linear_act_backward(dy.to(cuda), x.to(cuda), w.to(cuda), pre, act="gelu_erf")
    cdf = 0.5 * torch.erfc(-zd / 2 ** 0.5)
    mag = cdf + (slope - cdf).abs()
    bad = (dx[:, :1].double().cpu() - slope).abs() - (2 * h * slope.abs() + (1 + 2 * h) * mag * err + 2 * tiny)
    assert bool((bad <= 0).all()), z[bad[:, 0] > 0]
    assert abs(float(db[1]) - float(slope.sum())) <= float(rows * 4 * U * mag.sum() + (mag * err).sum() + h * slope.sum())
