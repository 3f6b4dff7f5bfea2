"""GPU: the norm's gradients of rows whose mean is large beside their spread.

Tolerance, with u = 2^-24, for the mean and rstd that the backward is given.  x - mean is one
rounding of the centred value, so xh = (x - mean) rstd errs by 2u |xh| however large the mean is.
dx = rstd (t - s1 - xh s2) rounds each of its three terms at most six times; the row sums s1 and s2 add at most
n = 40 + width / 512 terms one after another.  dw adds d xh over the rows: a CTA's own (rows / 148 at most),
16 lane groups, and 2960 lines in 128 groups of at most 24, a warp's tree over four of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("width", [64, 256, 515, 1022, 2056, 5120, 5121, 8200, 40000])
@pytest.mark.parametrize("ratio", [1e2, 1e3, 1e4])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_gradients_of_rows_far_from_zero(cuda, width, ratio, dtype):
    from vdn_b200.layer_norm import layer_norm, layer_norm_backward
    if dtype == torch.float16:
        ratio /= 10                                       # what 11 bits still resolve
    gen = torch.Generator().manual_seed(width)
    rows = 7
    noise = torch.randn(rows, width, generator=gen)
    x = (ratio * (1 + torch.rand(rows, 1, generator=gen)) + noise).to(dtype)
    dy = (noise + 0.3 * torch.randn(rows, width, generator=gen)).to(dtype)      # along x: s2 is near 1
    w = (1 + 0.2 * torch.randn(width, generator=gen)).float()
    _, mean, rstd = layer_norm(x.to(cuda), w.to(cuda), return_stats=True)
    dx, dw, db = layer_norm_backward(dy.to(cuda), x.to(cuda), w.to(cuda), mean, rstd)
    xd, d, wd = x.double(), dy.double(), w.double()
    m, r = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    xh, t = (xd - m) * r, d * wd
    s1, s2 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
    want = r * (t - s1 - xh * s2)
    n = 40 + width / 512
    e_s1, e_s2 = (n + 4) * U * t.abs().mean(1, keepdim=True), (n + 8) * U * (t * xh).abs().mean(1, keepdim=True)
    err = r * (6 * U * (t.abs() + s1.abs() + (xh * s2).abs()) + e_s1 + xh.abs() * e_s2)
    half = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    bad = (dx.double().cpu() - want).abs() - (err + half * (want.abs() + err) + tiny)
    assert bool((bad <= 0).all()), float((dx.double().cpu() - want).abs().max())
    chain = rows / 148 + 16 + 24 + 9
    err = (chain + 3) * U * (d * xh).abs().sum(0)
    assert bool(((dw.double().cpu() - (d * xh).sum(0)).abs() <= err + U * ((d * xh).sum(0).abs() + err)).all())
    err = chain * U * d.abs().sum(0)
    assert bool(((db.double().cpu() - d.sum(0)).abs() <= err + U * (d.sum(0).abs() + err)).all())
