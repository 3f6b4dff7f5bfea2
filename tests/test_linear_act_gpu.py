"""GPU: the linear layer with its epilogue, and its gradients, against 64-bit formulas.

Tolerances, with u = 2^-24 and h = eps/2 of the 16-bit type.  The tensor core adds k products
in fp32, in an order of its own, and may cut rather than round: an error of at most
(k + 16) 2u of the sum of magnitudes S = |x| |w|^T + |b|.  An activation has slope at most 1.13
and is itself computed to 2^-20 of its argument's magnitude.  y adds its one rounding.  In
the backward dz is rounded to 16 bits (h |dz|) before the products."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACTS = ["none", "gelu_tanh", "gelu_erf", "silu"]


def _half(t):
    return torch.finfo(t).eps / 2


def _tiny(t):
    return float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps / 2   # half the smallest step


def _act(z, act):
    """(value, slope) in 64 bits."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "gelu_erf":
        cdf = 0.5 * torch.erfc(-z / 2 ** 0.5)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    k = 2 * (2 / torch.pi) ** 0.5
    v = k * (z + 0.044715 * z ** 3) if act == "gelu_tanh" else z
    dv = k * (1 + 3 * 0.044715 * z * z) if act == "gelu_tanh" else torch.ones_like(z)
    p = torch.sigmoid(v)
    return z * p, p + z * dv * p * torch.sigmoid(-v)


def _inputs(seed, rows, n, k, dtype):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=gen).to(dtype)
    w = (torch.randn(n, k, generator=gen) * 1.5 * k ** -0.5).to(dtype)
    b = torch.randn(n, generator=gen).to(dtype)
    res, dy = (torch.randn(rows, n, generator=gen).to(dtype) for _ in range(2))
    return x, w, b, res, dy


def _wide(t, cuda):
    return None if t is None else t.to(cuda).double()


def _forward_check(cuda, x, w, b, res, act, y, pre):
    dtype = x.dtype
    h, tiny, k = _half(dtype), _tiny(dtype), x.shape[-1]
    xd, wd, bd, rd = (_wide(t, cuda) for t in (x, w, b, res))
    z = xd @ wd.T + (0 if b is None else bd)
    s = xd.abs() @ wd.abs().T + (0 if b is None else bd.abs())
    e = (k + 16) * 2 * U * s
    if pre is not None:
        assert bool(((pre.double() - z).abs() <= e + h * (z.abs() + e) + tiny).all())
    v, _ = _act(z, act)
    want = v + (0 if res is None else rd)
    err = 1.13 * e + 2.0 ** -20 * z.abs() + 2 * U * want.abs()
    bad = (y.double() - want).abs() > err + h * (want.abs() + err) + tiny
    assert not bool(bad.any()), (int(bad.sum()), float((y.double() - want).abs().max()))


def _backward_check(cuda, x, w, pre, dy, act, dx, dw, db):
    dtype = x.dtype
    h, tiny = _half(dtype), _tiny(dtype)
    rows, n, k = dy.shape[0], dy.shape[1], x.shape[1]
    xd, wd, d = _wide(x, cuda), _wide(w, cuda), _wide(dy, cuda)
    if act != "none":
        _, slope = _act(pre.double(), act)
        e_dz = d.abs() * (slope.abs() + pre.double().abs() + 1) * 2.0 ** -20 + tiny
        d = d * slope
    else:
        e_dz = torch.zeros_like(d)
    e_op = e_dz + (h * (d.abs() + e_dz) + tiny if act != "none" else 0)
    for got, want, mag, err, terms in ((dx, d @ wd, d.abs() @ wd.abs(), e_op @ wd.abs(), n),
                                       (dw, d.T @ xd, d.abs().T @ xd.abs(), e_op.T @ xd.abs(), rows)):
        err = err + (terms + 16) * 2 * U * mag
        bad = (got.double() - want).abs() > err + h * (want.abs() + err) + tiny
        assert not bool(bad.any()), (tuple(got.shape), int(bad.sum()), float((got.double() - want).abs().max()))
    if db is not None:
        want, mag = d.sum(0), d.abs().sum(0)
        err = e_dz.sum(0) + (rows / 512 + 96) * U * mag
        assert bool(((db.double() - want).abs() <= err + h * (want.abs() + err) + tiny).all())


def _both(cuda, seed, rows, n, k, dtype, act, bias=True, residual=True):
    from vdn_b200.linear_act import linear_act, linear_act_backward
    x, w, b, res, dy = _inputs(seed, rows, n, k, dtype)
    b, res = b if bias else None, res if residual else None
    dev = lambda t: None if t is None else t.to(cuda)
    y, pre = linear_act(dev(x), dev(w), dev(b), act=act, residual=dev(res), return_pre=True)
    plain = linear_act(dev(x), dev(w), dev(b), act=act, residual=dev(res))
    dx, dw, db = linear_act_backward(dev(dy), dev(x), dev(w), pre, act=act, bias=bias)
    torch.cuda.synchronize()
    assert y.dtype == dx.dtype == dw.dtype == dtype and y.shape == (rows, n)
    assert torch.equal(y, plain)
    _forward_check(cuda, x, w, b, res, act, y, pre)
    _backward_check(cuda, x, w, pre, dy, act, dx, dw, db)
    assert (db is None) == (not bias)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_activations_and_types(cuda, act, dtype):
    _both(cuda, 1, 300, 264, 200, dtype, act)


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 128, 64), (2, 130, 72), (16, 512, 1024), (17, 96, 640), (33, 777, 1004),
                                      (64, 256, 2048), (65, 129, 63), (128, 640, 129), (200, 1000, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_few_rows_and_odd_sizes(cuda, rows, n, k, dtype):
    _both(cuda, rows + n, rows, n, k, dtype, "gelu_tanh")


@pytest.mark.parametrize("rows,n,k,act,bias,residual", [
    (2048, 1024, 512, "none", True, True), (1801, 1100, 320, "gelu_tanh", True, False), (2000, 1025, 77, "silu", False, True),
    (1030, 2056, 1280, "none", False, False), (4100, 520, 64, "gelu_erf", True, True)])
def test_many_tiles(cuda, rows, n, k, act, bias, residual):
    """Outputs of 28 and more 256 x 256 tiles in the forward (and in the gradients' products)."""
    _both(cuda, rows, rows, n, k, torch.bfloat16, act, bias, residual)


def test_deep_sums(cuda):
    _both(cuda, 3, 40, 260, 13824, torch.bfloat16, "none")
    _both(cuda, 4, 9000, 136, 72, torch.float16, "silu")


def test_strided_operands_and_shapes(cuda):
    from vdn_b200.linear_act import linear_act, linear_act_backward
    x, w, b, res, dy = (t.to(cuda) for t in _inputs(5, 96, 160, 64, torch.bfloat16))
    want = linear_act(x, w, b, act="silu", residual=res)
    wide = torch.zeros(96, 400, dtype=torch.bfloat16, device=cuda)
    for off in (8, 3):
        wide[:, off:off + 64] = x
        wide[:, 100 + off:260 + off] = res
        assert torch.equal(linear_act(wide[:, off:off + 64], w, b, act="silu", residual=wide[:, 100 + off:260 + off]), want)
    wt = w.t().contiguous().t()
    assert torch.equal(linear_act(x, wt, b, act="silu", residual=res), want)
    assert torch.equal(linear_act(x.view(2, 3, 16, 64), w, b, act="silu", residual=res.view(2, 3, 16, 160)),
                       want.view(2, 3, 16, 160))
    assert torch.equal(linear_act(x[0], w, b), linear_act(x[:1], w, b)[0])
    row = res[:1].expand(96, 160)
    assert torch.equal(linear_act(x, w, b, residual=row), linear_act(x, w, b, residual=row.contiguous()))
    one = dy[:1].expand(96, 160)
    a, c = linear_act_backward(one, x, w), linear_act_backward(one.contiguous(), x, w)
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    flat = torch.zeros(96 * 160 + 1, dtype=torch.bfloat16, device=cuda)[1:].view(96, 160)   # 2-byte aligned
    flat.copy_(res)
    assert torch.equal(linear_act(x, w, b, act="silu", residual=flat), want)


def test_offsets_past_32_bits(cuda):
    from vdn_b200.linear_act import linear_act, linear_act_backward
    rows, n, k = 430000, 5120, 64
    x, w, b, _, _ = (t.to(cuda) for t in _inputs(6, 64, n, k, torch.bfloat16))
    big = torch.zeros(rows, k, dtype=torch.bfloat16, device=cuda)
    big[-64:] = x
    y, pre = linear_act(big, w, b, act="silu", return_pre=True)
    few, few_pre = linear_act(x, w, b, act="silu", return_pre=True)
    # two kernels, two orders of the sums: a rounding step of the result apart at most
    assert bool(((y[-64:].float() - few.float()).abs() <= 2.0 ** -7 * few.float().abs() + 1e-4).all())
    assert bool(((pre[-64:].float() - few_pre.float()).abs() <= 2.0 ** -7 * few_pre.float().abs() + 1e-4).all())
    del y
    dy = torch.zeros(rows, n, dtype=torch.bfloat16, device=cuda)
    dy[-64:] = few
    dx, dw, db = linear_act_backward(dy, big, w, pre, act="silu")
    ex, ew, eb = linear_act_backward(few, x, w, few_pre, act="silu")
    for p, q in ((dx[-64:], ex), (dw, ew), (db, eb)):
        assert float((p.float() - q.float()).norm()) <= 2.0 ** -6 * float(q.float().norm())
    assert not bool(dx[:-64].any())


def test_large_values(cuda):
    """Saturated activations: no NaN from overflowing exponentials or cubes."""
    from vdn_b200.linear_act import linear_act, linear_act_backward
    for dtype, top in ((torch.bfloat16, 1e30), (torch.float16, 6e4)):
        x = torch.zeros(4, 64, dtype=dtype, device=cuda)
        x[:, 0] = torch.tensor([top, -top, 20.0, -20.0])
        w = torch.zeros(32, 64, dtype=dtype, device=cuda)
        w[:, 0] = 1
        for act in ACTS:
            y, pre = linear_act(x, w, act=act, return_pre=True)
            want = _act(x[:, :1].double().clamp(-200, 200), act)[0]
            want = torch.where(x[:, :1].double().abs() > 200, x[:, :1].double() if act == "none" else
                               x[:, :1].double().clamp(min=0), want)
            err = _half(dtype) * want.abs() + 2.0 ** -20 * 20 + _tiny(dtype)
            assert bool(((y.double() - want).abs() <= err).all()), act
            dx, dw, db = linear_act_backward(torch.ones_like(y), x, w, pre, act=act)
            slope = torch.tensor([1.0, 1.0 if act == "none" else 0.0], device=cuda).double()
            assert bool(torch.isfinite(dx).all())
            assert bool(((dx[:2, 0].double() - 32 * slope).abs() <= 32 * 2.0 ** -8).all()), act


def test_same_bits_streams_and_graphs(cuda):
    from vdn_b200.linear_act import linear_act, linear_act_backward
    x, w, b, res, dy = (t.to(cuda) for t in _inputs(7, 700, 512, 256, torch.bfloat16))

    def both():
        y, pre = linear_act(x, w, b, act="gelu_tanh", residual=res, return_pre=True)
        few = linear_act(x[:20], w, b)
        return (y, few, *linear_act_backward(dy, x, w, pre, act="gelu_tanh"))
    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    here = both()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, other, here))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(both())
            with pytest.raises(RuntimeError, match="capture"):
                linear_act(x.clone().requires_grad_(), w, b)
    x.mul_(0.5)
    want = both()
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(want, *outs))


@pytest.mark.parametrize("act", ACTS)
def test_autograd_matches_the_explicit_backward(cuda, act):
    from vdn_b200.linear_act import linear_act, linear_act_backward
    x, w, b, res, dy = (t.to(cuda) for t in _inputs(8, 70, 96, 64, torch.bfloat16))
    leaves = [t.clone().requires_grad_() for t in (x, w, b, res)]
    y = linear_act(leaves[0], leaves[1], leaves[2], act=act, residual=leaves[3])
    y.backward(dy)
    y2, pre = linear_act(x, w, b, act=act, residual=res, return_pre=True)
    want = (*linear_act_backward(dy, x, w, pre, act=act), dy)
    assert torch.equal(y, y2) and all(torch.equal(leaf.grad, g) for leaf, g in zip(leaves, want))
    only = b.clone().requires_grad_()
    linear_act(x, w, only, act=act).backward(dy)
    assert torch.equal(only.grad, want[2])


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(cuda, act):
    """The gradients along random directions against central differences of the formula in
    64 bits, at points that 16 bits hold exactly; h covers dz, pre and the outputs."""
    from vdn_b200.linear_act import linear_act, linear_act_backward
    x, w, b, _, dy = _inputs(9, 24, 40, 48, torch.float16)
    y, pre = linear_act(x.to(cuda), w.to(cuda), b.to(cuda), act=act, return_pre=True)
    grads = linear_act_backward(dy.to(cuda), x.to(cuda), w.to(cuda), pre, act=act)

    def loss(xv, wv, bv):
        return (_act(xv @ wv.T + bv, act)[0] * dy.double()).sum()
    base = [t.double() for t in (x, w, b)]
    gen = torch.Generator().manual_seed(2)
    # every gradient is a sum of d_ij c_ij: dz errs by h |dz| (rounding), h |pre| |act''| |dy| (pre's
    # rounding, |act''| <= 1.2) and each result by h of itself
    z = base[0] @ base[1].T + base[2]
    e_dz = 2.0 ** -11 * dy.double().abs() * (1.13 + 1.2 * z.abs()) + 1e-6
    spans = [e_dz @ base[1].abs(), e_dz.T @ base[0].abs(), e_dz.sum(0)]
    for i, (g, span) in enumerate(zip(grads, spans)):
        way = torch.randn(base[i].shape, generator=gen).double()
        diff = (loss(*[v + 1e-5 * way if j == i else v for j, v in enumerate(base)])
                - loss(*[v - 1e-5 * way if j == i else v for j, v in enumerate(base)])) / 2e-5
        got = g.double().cpu()
        limit = ((span + 2.0 ** -11 * got.abs()) * way.abs()).sum() * 1.01 + 1e-4
        assert abs(float((got * way).sum() - diff)) <= float(limit), i


def test_refusals_and_empty(cuda):
    from vdn_b200.linear_act import linear_act, linear_act_backward
    x = torch.zeros(4, 16, dtype=torch.bfloat16, device=cuda)
    w = torch.zeros(8, 16, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(TypeError, match="both"):
        linear_act(x, w.half())
    with pytest.raises(TypeError, match="both"):
        linear_act(x.float(), w.float())
    with pytest.raises(ValueError, match="weight"):
        linear_act(x[:, :8], w)
    with pytest.raises(ValueError, match="act"):
        linear_act(x, w, act="relu")
    with pytest.raises(ValueError, match="bias"):
        linear_act(x, w, torch.zeros(9, dtype=torch.bfloat16, device=cuda))
    with pytest.raises(ValueError, match="residual"):
        linear_act(x, w, residual=torch.zeros(4, 9, dtype=torch.bfloat16, device=cuda))
    with pytest.raises(ValueError, match="pre"):
        linear_act_backward(torch.zeros(4, 8, dtype=torch.bfloat16, device=cuda), x, w, act="silu")
    y, pre = linear_act(x[:0], w, act="silu", return_pre=True)
    dx, dw, db = linear_act_backward(y, x[:0], w, pre, act="silu")
    assert y.shape == (0, 8) and dx.shape == (0, 16) and not bool(dw.any()) and not bool(db.any())
