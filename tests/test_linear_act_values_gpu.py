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
