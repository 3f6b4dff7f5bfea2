"""GPU: layer norm and its gradients against the formulas in 64 bits.

Tolerances, with u = 2^-24.  A row sum adds at most n = 40 + width / 512 terms one after
another (registers, lanes, warps), so it errs by n u of the sum of magnitudes; the value
itself and each factor round once or twice.  An output rounds by eps/2."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
PAIRS = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.float32, torch.float32)]


def _half(t):
    return torch.finfo(t).eps / 2


def _inputs(seed, rows, width, dtype, w_dtype):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, width, generator=gen) * 2 + torch.randn(rows, 1, generator=gen) * 3).to(dtype)
    w = (1 + 0.2 * torch.randn(width, generator=gen)).to(w_dtype)
    b = (0.5 * torch.randn(width, generator=gen)).to(w_dtype)
    dy = torch.randn(rows, width, generator=gen).to(dtype)
    return x, w, b, dy


def _check(cuda, x, w, b, dy, eps=1e-5):
    from vdn_b200.layer_norm import layer_norm, layer_norm_backward
    dev = lambda t: None if t is None else t.to(cuda)
    rows, width = x.shape
    y, mean, rstd = layer_norm(dev(x), dev(w), dev(b), eps, return_stats=True)
    n = 40 + width / 512
    xd = x.double()
    mu = xd.mean(1, keepdim=True)
    r = 1 / torch.sqrt((xd - mu).square().mean(1, keepdim=True) + eps)
    wd = w.double() if w is not None else torch.ones(width, dtype=torch.float64)
    bd = b.double() if b is not None else torch.zeros(width, dtype=torch.float64)
    want = (xd - mu) * r * wd + bd
    e_mu = n * U * xd.abs().mean(1, keepdim=True) + 2 * U * mu.abs()
    # the mean's error moves the centred values (and the variance by its square only)
    e_r = (n + 8) * U + (e_mu * r).square()
    err = wd.abs() * r * (e_mu + U * (xd - mu).abs()) + (want - bd).abs() * (e_r + 4 * U) + U * want.abs()
    got = y.double().cpu()
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    assert y.dtype == x.dtype and y.shape == x.shape
    assert bool(((got - want).abs() <= err + _half(x.dtype) * (want.abs() + err) + tiny).all())
    assert bool(((mean.double().cpu()[:, None] - mu).abs() <= e_mu).all())
    assert bool(((rstd.double().cpu()[:, None] - r).abs() <= r * (e_r + 4 * U)).all())

    grads = layer_norm_backward(dev(dy), dev(x), dev(w), mean, rstd, bias=b is not None)
    m1, r1 = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]     # what the backward is given
    d = dy.double()
    xh, t = (xd - m1) * r1, d * wd
    s1, s2 = t.mean(1, keepdim=True), (t * xh).mean(1, keepdim=True)
    dx = r1 * (t - s1 - xh * s2)
    e_s1, e_s2 = (n + 4) * U * t.abs().mean(1, keepdim=True), (n + 8) * U * (t * xh).abs().mean(1, keepdim=True)
    e_xh = 3 * U * (xd.abs() + m1.abs()) * r1
    err = r1 * (4 * U * (t.abs() + s1.abs() + (xh * s2).abs()) + e_s1 + xh.abs() * e_s2 + e_xh * s2.abs())
    got = grads[0].double().cpu()
    assert grads[0].dtype == x.dtype
    assert bool(((got - dx).abs() <= err + _half(x.dtype) * (dx.abs() + err) + tiny).all())
    chain = rows / 296 + 16 + 2960 / 32 + 32      # rows of one CTA, its lane groups, at most 2960 lines in 32 groups
    for got, want, mag, extra, on in ((grads[1], (d * xh).sum(0), (d * xh).abs().sum(0), (d.abs() * e_xh).sum(0), w is not None),
                                      (grads[2], d.sum(0), d.abs().sum(0), 0.0, b is not None)):
        if not on:
            assert got is None
            continue
        kind = (w if w is not None else x).dtype
        assert got.dtype == kind and got.shape == (width,)
        err = (chain + 2) * U * mag + extra
        assert bool(((got.double().cpu() - want).abs() <= err + _half(kind) * (want.abs() + err)).all())
    return y, grads


@pytest.mark.parametrize("dtype,w_dtype", PAIRS)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (5, 64), (33, 128), (4, 130), (300, 256), (7, 512), (9, 777),
                                        (2, 1024), (11, 2056), (40, 5120), (3, 5121), (2, 8200), (2, 16384), (2, 40000)])
def test_types_and_widths(cuda, dtype, w_dtype, rows, width):
    x, w, b, dy = _inputs(rows + width, rows, width, dtype, w_dtype)
    _check(cuda, x, w, b, dy)


@pytest.mark.parametrize("rows,width", [(2000, 64), (1201, 320), (700, 1024), (650, 6152), (900, 33)])
def test_many_rows(cuda, rows, width):
    x, w, b, dy = _inputs(rows, rows, width, torch.bfloat16, torch.float32)
    _check(cuda, x, w, b, dy)


@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_optional_parameters(cuda, has_w, has_b):
    x, w, b, dy = _inputs(5, 30, 200, torch.float16, torch.float16)
    _check(cuda, x, w if has_w else None, b if has_b else None, dy)


def test_constant_rows_and_extremes(cuda):
    """No variance: the result is the bias; values near the type's limits stay finite."""
    from vdn_b200.layer_norm import layer_norm
    x = torch.full((4, 96), 3.0, dtype=torch.bfloat16, device=cuda)
    b = torch.arange(96, device=cuda).bfloat16()
    assert torch.equal(layer_norm(x, None, b), b.expand(4, 96))
    big = torch.full((2, 512), 60000.0, dtype=torch.float16, device=cuda)
    big[:, ::2] = -60000.0
    y = layer_norm(big)
    assert torch.equal(y.float().abs(), torch.ones_like(y).float())
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    y = layer_norm(x)
    assert bool(torch.isfinite(y[[0, 3]]).all()) and bool(torch.isnan(y[1]).all())


def test_strides_shapes_and_expanded_gradients(cuda):
    from vdn_b200.layer_norm import layer_norm, layer_norm_backward
    x, w, b, dy = (t.to(cuda) for t in _inputs(6, 24, 128, torch.bfloat16, torch.bfloat16))
    want = layer_norm(x, w, b)
    wide = torch.zeros(24, 300, dtype=torch.bfloat16, device=cuda)
    for off in (0, 8, 3):                                  # aligned, and not
        wide[:, off:off + 128] = x
        assert float((layer_norm(wide[:, off:off + 128], w, b).float() - want.float()).abs().max()) <= 2.0 ** -6
    assert torch.equal(layer_norm(x.view(2, 3, 4, 128), w, b), want.view(2, 3, 4, 128))
    turned = x.t().contiguous().t()
    assert torch.equal(layer_norm(turned, w, b), want)
    _, mean, rstd = layer_norm(x, w, b, return_stats=True)
    one = dy[:1].expand(24, 128)                           # one gradient row for all
    got = layer_norm_backward(one, x, w, mean, rstd)
    ref = layer_norm_backward(one.contiguous(), x, w, mean, rstd)
    assert all(torch.equal(p, q) for p, q in zip(got, ref))
    assert torch.equal(layer_norm(x[0], w, b), want[0])


def test_same_bits_streams_and_graphs(cuda):
    from vdn_b200.layer_norm import layer_norm, layer_norm_backward
    x, w, b, dy = (t.to(cuda) for t in _inputs(7, 3000, 640, torch.bfloat16, torch.float32))

    def both():
        y, mean, rstd = layer_norm(x, w, b, return_stats=True)
        return (y, *layer_norm_backward(dy, x, w, mean, rstd))
    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    here = both()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, other, here))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]    # two graphs, workspaces of their own
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(both())
            with pytest.raises(RuntimeError, match="capture"):
                layer_norm(x.clone().requires_grad_(), w, b)
    x.add_(dy)
    want = both()
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, *outs))


def test_offsets_past_32_bits(cuda):
    from vdn_b200.layer_norm import layer_norm, layer_norm_backward
    rows, width = 430000, 5120
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(1)
    x[-40:] = torch.randn(40, width, generator=gen, device=cuda).bfloat16()
    w = torch.rand(width, generator=gen, device=cuda)
    y, mean, rstd = layer_norm(x, w, w, return_stats=True)
    assert torch.equal(y[-40:], layer_norm(x[-40:], w, w)) and torch.equal(y[:2], w.bfloat16().expand(2, width))
    dx, dw, db = layer_norm_backward(x, x, w, mean, rstd)
    ex, ew, eb = layer_norm_backward(x[-40:], x[-40:], w, mean[-40:], rstd[-40:])
    assert torch.equal(dx[-40:], ex) and not bool(dx[:-40].any())
    assert bool(((dw - ew).abs() <= 64 * U * (ew.abs() + 40)).all()) and bool(((db - eb).abs() <= 64 * U * 200).all())


def test_gradients_against_differences(cuda):
    from vdn_b200.layer_norm import layer_norm
    gen = torch.Generator().manual_seed(1)
    x, w, b = torch.randn(6, 48, generator=gen), torch.randn(48, generator=gen), torch.randn(48, generator=gen)
    weight = torch.randn(6, 48, generator=gen).double()

    def loss(xv, wv, bv):
        m = xv.mean(1, keepdim=True)
        return (((xv - m) / torch.sqrt((xv - m).square().mean(1, keepdim=True) + 1e-5) * wv + bv) * weight).sum()
    leaves = [t.to(cuda).requires_grad_() for t in (x, w, b)]
    (layer_norm(*leaves) * weight.to(cuda).float()).sum().backward()
    base = [t.double() for t in (x, w, b)]
    for k, leaf in enumerate(leaves):
        way = torch.randn(base[k].shape, generator=gen).double()
        diff = (loss(*[v + 1e-5 * way if i == k else v for i, v in enumerate(base)])
                - loss(*[v - 1e-5 * way if i == k else v for i, v in enumerate(base)])) / 2e-5
        terms = leaf.grad.double().cpu() * way
        assert abs(float(terms.sum() - diff)) < 1e-5 * float(terms.abs().sum()), k


def test_refusals_and_empty(cuda):
    from vdn_b200.layer_norm import layer_norm, layer_norm_backward
    x = torch.zeros(4, 16, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(TypeError, match="weight"):
        layer_norm(x, torch.ones(16, device=cuda, dtype=torch.float16))
    with pytest.raises(ValueError, match="weight"):
        layer_norm(x, torch.ones(17, device=cuda))
    with pytest.raises(TypeError, match="share"):
        layer_norm(x, torch.ones(16, device=cuda), torch.ones(16, device=cuda).bfloat16())
    with pytest.raises(ValueError, match="grad_y"):
        layer_norm_backward(x.float(), x, None, torch.zeros(4, device=cuda), torch.zeros(4, device=cuda))
    with pytest.raises(ValueError, match="mean"):
        layer_norm_backward(x, x, None, torch.zeros(3, device=cuda), torch.zeros(4, device=cuda))
    none = x[:0]
    w = torch.ones(16, device=cuda)
    y, mean, rstd = layer_norm(none, w, return_stats=True)
    dx, dw, db = layer_norm_backward(none, none, w, mean, rstd)
    assert y.shape == dx.shape == (0, 16) and not bool(dw.any()) and not bool(db.any())
