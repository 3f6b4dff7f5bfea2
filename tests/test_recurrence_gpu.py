"""GPU: the gated scan and its gradients against the recurrence in 64 bits.

Tolerance.  With u = 2^-24, each step rounds its sum (2u |h_t|) and uses a decay within
5u of exp(g) (the hardware exponential's 2^-22 and a rounding), so it adds at most 8u M_t, where M is the same recurrence on absolute values.  An
error then decays like the state: the total is at most 8u E_t with E the recurrence fed
with M.  The output's own rounding adds eps/2 |y_t|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _scan(a, x, h0):
    """h over dim 0 in 64 bits; the states before each step as well."""
    out, h = [], h0
    before = []
    for t in range(x.shape[0]):
        before.append(h)
        h = a[t] * h + x[t]
        out.append(h)
    stack = (lambda v: torch.stack(v)) if out else (lambda v: x.new_zeros(x.shape))
    return stack(out), stack(before), h


def _reference(x, g, h0, dy, dlast, y_saved):
    """Of one sequence [T, C], all in 64 bits: outputs, gradients and their bounds."""
    a = g.exp()
    y, _, last = _scan(a, x, h0)
    m, _, ml = _scan(a, x.abs(), h0.abs())
    e, _, el = _scan(a, m, torch.zeros_like(h0))
    res = dict(y=y, last=last, y_err=8 * U * e, last_err=8 * U * el)
    if dy is None:
        return res
    before = torch.cat([h0[None], y_saved[:-1]]) if len(x) else y_saved
    af = a.flip(0)

    def back(v, c):
        us = []
        for t in range(len(v)):
            us.append(v[t] + c)
            c = af[t] * us[-1]
        return (torch.stack(us) if us else v.new_zeros(v.shape)), c
    u, ds = back(dy.flip(0), dlast)
    mu, mds = back(dy.flip(0).abs(), dlast.abs())
    eu, eds = back(mu, torch.zeros_like(dlast))
    u, mu, eu = u.flip(0), mu.flip(0), eu.flip(0)
    res.update(dx=u, dx_err=8 * U * eu, ds=ds, ds_err=8 * U * eds, dg=a * u * before,
               dg_err=16 * U * a * (eu + mu) * before.abs())
    return res


def _close(got, want, err, what):
    got = got.double().cpu()
    bad = (got - want).abs() > err
    assert not bool(bad.any()), (what, [(float(g), float(w), float(e)) for g, w, e in
                                        zip(got[bad][:4], want[bad][:4], err[bad][:4])])


def _half(t):
    return torch.finfo(t).eps / 2


def _case(seed, lead, h, d, dtype, g_dtype, shared, sharp=False):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(*lead, h, d, generator=gen).to(dtype)
    shape = (*lead, h) if shared else (*lead, h, d)
    g = -torch.exp(torch.rand(shape, generator=gen) * 9 - 8)
    if sharp:                                             # restarts and strong decays among slow ones
        pick = torch.rand(shape, generator=gen)
        g = torch.where(pick < 0.1, torch.full_like(g, -float("inf")), torch.where(pick < 0.3, g * 30, g))
    return gen, x, g.to(g_dtype)


def _run(cuda, x, g, cu, reverse, with_state, gen, back=True):
    """Compares gated_scan and gated_scan_backward with the reference, sequence by sequence."""
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    dtype, gd = x.dtype, g.dtype
    packed = cu is not None
    seqs = len(cu) - 1 if packed else x.shape[0]
    tail = x.shape[1:] if packed else x.shape[2:]
    state = torch.randn(seqs, *tail, generator=gen) if with_state else None
    dlast = torch.randn(seqs, *tail, generator=gen) if with_state else None
    dy = torch.randn(x.shape, generator=gen).to(dtype)
    dev = lambda t: None if t is None else t.to(cuda)
    cud = torch.tensor(cu, dtype=torch.int32, device=cuda) if packed else None
    y, last = gated_scan(dev(x), dev(g), dev(state), cu_seqlens=cud, reverse=reverse)
    got_back = gated_scan_backward(dev(dy), dev(g), y, state=dev(state), grad_state=dev(dlast), cu_seqlens=cud,
                                   reverse=reverse) if back else None
    torch.cuda.synchronize()
    assert y.dtype == dtype and last.dtype == torch.float32
    shared = g.dim() < x.dim()
    # Below a type's normal range its step is smallest_normal * eps, so a result that lies there
    # rounds by up to half of that (fp16: 2^-14 * 2^-10 / 2 = 2^-25), however small it is.
    tiny = lambda t: float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps / 2
    for s in range(seqs):
        rows = slice(cu[s], cu[s + 1]) if packed else slice(None)
        pick = (lambda t: t[rows]) if packed else (lambda t: t[s])
        turn = (lambda t: t.flip(0)) if reverse else (lambda t: t)
        gs = turn(pick(g)).double()
        gs = (gs[..., None].expand(*gs.shape, x.shape[-1]) if shared else gs)
        flat = lambda t: turn(pick(t)).double().cpu().flatten(1)
        zero = torch.zeros(tail.numel(), dtype=torch.float64)
        h0 = state[s].double().flatten() if with_state else zero
        ref = _reference(flat(x), gs.flatten(1), h0, flat(dy) if back else None,
                         dlast[s].double().flatten() if with_state else zero, flat(y) if back else None)
        _close(flat(y), ref["y"], ref["y_err"] + _half(dtype) * (ref["y"].abs() + ref["y_err"]) + tiny(dtype), "y")
        _close(last[s].flatten(), ref["last"], ref["last_err"] + U * ref["last"].abs(), "last")
        if not back:
            continue
        dx, dg, ds = got_back
        assert dx.dtype == dtype and dg.dtype == gd and ds.dtype == torch.float32
        _close(flat(dx), ref["dx"], ref["dx_err"] + _half(dtype) * (ref["dx"].abs() + ref["dx_err"]) + tiny(dtype), "dx")
        _close(ds[s].flatten(), ref["ds"], ref["ds_err"] + U * ref["ds"].abs(), "ds")
        want, err = ref["dg"], ref["dg_err"]
        if shared:                                        # a sum of d terms, in a tree of at most 9 levels
            n = want.shape[0]
            err = (err + 9 * U * want.abs()).view(n, x.shape[-2], x.shape[-1]).sum(-1)
            want = want.view(n, x.shape[-2], x.shape[-1]).sum(-1)
            gotg = turn(pick(dg)).double().cpu()
        else:
            gotg = flat(dg)
        _close(gotg, want, err + _half(gd) * (want.abs() + err) + tiny(gd), "dg")
    return y, got_back


TYPES = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
         (torch.float16, torch.float32), (torch.float32, torch.float32)]


@pytest.mark.parametrize("dtype,g_dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 2, 7, 64, 65, 1001])
def test_dense_types_and_lengths(cuda, dtype, g_dtype, tokens):
    gen, x, g = _case(tokens, (2, tokens), 3, 40, dtype, g_dtype, False)
    _run(cuda, x, g, None, tokens % 2 == 0, True, gen)


@pytest.mark.parametrize("heads,d", [(1, 1), (1, 31), (1, 33), (5, 13), (2, 64), (1, 515)])
@pytest.mark.parametrize("reverse", [False, True])
def test_dense_odd_widths(cuda, heads, d, reverse):
    gen, x, g = _case(d, (3, 130), heads, d, torch.bfloat16, torch.float32, False)
    _run(cuda, x, g, None, reverse, heads % 2 == 0, gen)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype,g_dtype", TYPES)
def test_shared_decay(cuda, d, dtype, g_dtype):
    gen, x, g = _case(d, (2, 300), 3, d, dtype, g_dtype, True)
    _run(cuda, x, g, None, d == 64, True, gen)


@pytest.mark.parametrize("cu", [[0, 5, 5, 70, 71, 400], [0, 0, 0], [0, 1], [3, 3, 9, 40], [0, 9, 600, 640]])
@pytest.mark.parametrize("shared,reverse", [(False, False), (True, True)])
def test_packed_lengths(cuda, cu, shared, reverse):
    """Empty sequences, sequences of one token, rows in front of the first and behind the last."""
    gen, x, g = _case(len(cu), (700,), 2, 64, torch.bfloat16, torch.float32, shared)
    y, (dx, dg, _) = _run(cuda, x, g, cu, reverse, True, gen)
    for t in (y, dx, dg):
        assert bool((t[cu[-1]:] == 0).all())


@pytest.mark.parametrize("dtype,g_dtype", TYPES)
@pytest.mark.parametrize("tokens,reverse", [(1024, False), (1025, True), (1499, False)])
def test_long_runs(cuda, dtype, g_dtype, tokens, reverse):
    """Few tiles and long sequences take 32 tokens a warp: whole and ragged last runs, sharp decays."""
    gen, x, g = _case(tokens, (1, tokens), 2, 36, dtype, g_dtype, False, sharp=True)
    _run(cuda, x, g, None, reverse, True, gen)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dtype,g_dtype", [TYPES[0], TYPES[3], TYPES[4]])
@pytest.mark.parametrize("tokens,reverse", [(1024, True), (1057, False)])
def test_long_runs_of_shared_decays(cuda, d, dtype, g_dtype, tokens, reverse):
    gen, x, g = _case(tokens + d, (1, tokens), 2, d, dtype, g_dtype, True, sharp=True)
    _run(cuda, x, g, None, reverse, True, gen)


def test_long_runs_of_shared_decays_packed(cuda):
    gen, x, g = _case(32, (4200,), 1, 128, torch.bfloat16, torch.float32, True)
    _run(cuda, x, g, [0, 1, 1100, 1100, 4100], False, True, gen)


def test_long_runs_packed_and_strided(cuda):
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    gen, x, g = _case(31, (4200,), 1, 64, torch.bfloat16, torch.bfloat16, False)
    _run(cuda, x, g, [0, 1, 1100, 1100, 4100], True, True, gen)
    x, g = x[:, 0].to(cuda), g[:, 0].to(cuda)
    y, last = gated_scan(x[None], g[None])
    back = gated_scan_backward(x[None], g[None], y)
    buf = torch.zeros(4200, 3, 66, dtype=torch.bfloat16, device=cuda)   # pairs aligned, tiles not
    buf[:, 0, 2:], buf[:, 1, 2:], buf[:, 2, 2:] = x, g, y[0]
    xs, gs, ys = (buf[:, i, 2:][None] for i in range(3))
    for a, b in zip((*gated_scan(xs, gs), *gated_scan_backward(xs, gs, ys)), (y, last, *back)):
        assert torch.equal(a, b)
    buf = torch.zeros(4200, 3, 67, dtype=torch.bfloat16, device=cuda)   # odd rows: single channels a lane
    buf[:, 0, 1:65], buf[:, 1, 1:65], buf[:, 2, 1:65] = x, g, y[0]
    xs, gs, ys = (buf[:, i, 1:65][None] for i in range(3))
    flat = lambda t: t.double().cpu()
    zero = torch.zeros(64, dtype=torch.float64)
    ref = _reference(flat(x), flat(g), zero, flat(x), zero, flat(y[0]))
    half = _half(torch.bfloat16)
    dx, dg, _ = gated_scan_backward(xs, gs, ys)
    for name, got in (("y", gated_scan(xs, gs)[0]), ("dx", dx), ("dg", dg)):
        _close(got[0], ref[name], ref[name + "_err"] + half * (ref[name].abs() + ref[name + "_err"]) + 2.0 ** -134, name)


@pytest.mark.parametrize("seqs", [2, 31, 32, 33])
def test_packed_order(cuda, seqs):
    """Up to 32 packed sequences start longest first: equal lengths, empty ones, the longest last."""
    lengths = [(7 * i) % 5 * 3 for i in range(seqs - 1)] + [90]
    cu = [2]
    for n in lengths:
        cu.append(cu[-1] + n)
    gen, x, g = _case(seqs, (cu[-1] + 5,), 1, 64, torch.bfloat16, torch.float32, False)
    y, (dx, dg, _) = _run(cuda, x, g, cu, False, True, gen)
    for t in (y, dx, dg):
        assert bool((t[cu[-1]:] == 0).all()) and bool((t[:cu[0]] == 0).all())


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("cu", [[300, 300], [40, 90, 300], [-5, 17, 900]])
def test_rows_outside_the_sequences_come_back_zero(cuda, shared, cu):
    """In front of the first sequence as behind the last; offsets out of range are cut off."""
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    gen, x, g = _case(41, (420,), 2, 64, torch.bfloat16, torch.float32, shared)
    x, g = x.to(cuda), g.to(cuda)
    cud = torch.tensor(cu, dtype=torch.int32, device=cuda)
    for _ in range(2):                                       # the second time over memory that held NaN
        y, _ = gated_scan(x, g, cu_seqlens=cud)
        dx, dg, _ = gated_scan_backward(x, g, y, cu_seqlens=cud)
        for t in (y, dx, dg):
            for part in (t[:max(cu[0], 0)], t[cu[-1]:]):
                assert bool((part == 0).all())
            t.fill_(float("nan"))
        del y, dx, dg, t, part
    out = torch.full_like(x, 5.0)
    gated_scan(x, g, cu_seqlens=cud, out=out)
    assert bool((out[:max(cu[0], 0)] == 5).all()) and bool((out[cu[-1]:] == 5).all())


@pytest.mark.parametrize("dtype,g_dtype", TYPES)
def test_restarts_and_strong_decays(cuda, dtype, g_dtype):
    """log_decay = -inf starts a channel anew, next to decays close to 1."""
    gen, x, g = _case(11, (1, 500), 2, 48, dtype, g_dtype, False, sharp=True)
    _run(cuda, x, g, None, False, True, gen)


def test_constant_slow_decay_keeps_its_memory(cuda):
    """A decay 2^-14 below 1 over 60000 tokens: rounding exp(g) to fp32 would shift the
    stationary state by up to 2^14 * 2^-25 = 5e-4 of itself.  Here the long chain joins runs of
    64 tokens: each join rounds the run's decay and the state once (2^-25 relative each, the
    decay and the state lying just below a power of two), the state remembers 16400 / 64
    joins, and a run's own fold errs by at most 16 * 2^-24: 256.25 * 2^-24 + 2^-20 = 1.63e-5."""
    from vdn_b200.recurrence import gated_scan
    n, c = 60000, 64
    g = torch.full((1, n, c), -1.0 / 16400)
    x = torch.ones(1, n, c)
    _, last = gated_scan(x.to(cuda), g.to(cuda))
    a = g[0, 0, 0].double().exp()
    want = (1 - a ** n) / (1 - a)
    assert float((last.double().cpu() - want).abs().max() / want) < 1.63e-5


def test_long_lengths_join_every_level(cuda):
    gen, x, g = _case(5, (1, 9000), 1, 32, torch.float32, torch.float32, False)
    _run(cuda, x, g, None, False, True, gen)
    gen, x, g = _case(6, (4500,), 1, 64, torch.bfloat16, torch.bfloat16, True)
    _run(cuda, x, g, [0, 4400, 4499], True, False, gen)


def test_strides_broadcast_and_outputs(cuda):
    from vdn_b200.recurrence import gated_scan
    gen, x, g = _case(3, (2, 90), 4, 32, torch.bfloat16, torch.bfloat16, False)
    want, last = gated_scan(x.to(cuda), g.to(cuda))
    fused = torch.zeros(2, 90, 3 * 128 + 2, dtype=torch.bfloat16, device=cuda)   # columns of one projection
    fused[..., 2:130], fused[..., 130:258] = x.to(cuda).flatten(2), g.to(cuda).flatten(2)
    xs, gs = fused[..., 2:130].unflatten(2, (4, 32)), fused[..., 130:258].unflatten(2, (4, 32))
    buf = torch.full((2, 90, 300), 7.0, dtype=torch.bfloat16, device=cuda)
    out = buf[..., 1:129].unflatten(2, (4, 32))
    state = torch.zeros(2, 4, 32, device=cuda)
    y, st = gated_scan(xs, gs, state, out=out, out_state=state)
    assert y is out and st is state
    assert torch.equal(out, want) and torch.equal(state, last)
    assert bool((buf[..., 0] == 7).all()) and bool((buf[..., 129:] == 7).all())
    turned = x.to(cuda).transpose(2, 3).contiguous().transpose(2, 3)               # channels not contiguous
    assert torch.equal(gated_scan(turned, g.to(cuda))[0], want)
    const = g[0, 0].to(cuda)
    wide = const.expand(2, 90, 4, 32)
    assert torch.equal(gated_scan(x.to(cuda), wide)[0], gated_scan(x.to(cuda), wide.contiguous())[0])


@pytest.mark.parametrize("d", [64, 128])
def test_shared_decay_of_misaligned_rows(cuda, d):
    """Rows that start inside a lane's vector are copied; an `out` like that is refused."""
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    gen, x, g = _case(d, (2, 40), 2, d, torch.bfloat16, torch.float32, True)
    x, g = x.to(cuda), g.to(cuda)
    y, last = gated_scan(x, g)
    want = (y, last, *gated_scan_backward(x, g, y))
    wide = torch.zeros(2, 40, 2 * d + 3, dtype=torch.bfloat16, device=cuda)
    flat = torch.zeros(x.numel() + 1, dtype=torch.bfloat16, device=cuda)[1:].view(x.shape)   # contiguous
    for view in (wide[..., 1:2 * d + 1].unflatten(2, (2, d)), flat):
        def put(t):
            view.copy_(t)
            return view
        got = gated_scan(put(x), g)
        for a, b in zip((*got, *gated_scan_backward(put(x), g, y), *gated_scan_backward(x, g, put(y))),
                        (*want, *want[2:])):
            assert torch.equal(a, b)
    with pytest.raises(ValueError, match="aligned"):
        gated_scan(x, g, out=flat)


def test_packed_out_keeps_rows_behind_the_last(cuda):
    from vdn_b200.recurrence import gated_scan
    gen, x, g = _case(4, (50,), 2, 32, torch.bfloat16, torch.bfloat16, True)
    out = torch.full_like(x, 3.0).to(cuda)
    gated_scan(x.to(cuda), g.to(cuda), cu_seqlens=torch.tensor([0, 20, 44], dtype=torch.int32, device=cuda), out=out)
    assert bool((out[44:] == 3).all()) and not bool((out[:44] == 3).all())


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("reverse", [False, True])
def test_rows_outside_the_sequences_do_not_matter(cuda, shared, reverse):
    """NaN and infinities in front of the first sequence and behind the last."""
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    gen, x, g = _case(21, (500,), 2, 64, torch.bfloat16, torch.bfloat16, shared)
    cu = torch.tensor([70, 75, 300, 431], dtype=torch.int32, device=cuda)
    x, g = x.to(cuda), g.to(cuda)

    def both():
        y, last = gated_scan(x, g, cu_seqlens=cu, reverse=reverse)
        return (y[70:431].clone(), last, *[t[70:431].clone() if t.dim() == x.dim() or t.shape == g.shape else t
                                           for t in gated_scan_backward(x, g, y, cu_seqlens=cu, reverse=reverse)])
    want = both()
    for t in (x, g):
        t[:70], t[431:] = float("nan"), float("inf")
    got = both()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(bool(torch.isfinite(t).all()) for t in got)


def test_offsets_past_32_bits(cuda):
    """2.2e9 elements: the last rows equal a scan of their own from the state before them.  The two
    group the sums differently, so each side errs by 8u E (|x| < 5, decay 0.78: M < 23, E < 105:
    5e-5) before its own rounding to bf16 by 2^-8 of the value: 2^-7 |value| + 1e-4 apart at most.
    In the backward |h| < 23 multiplies the fp32 part for dg."""
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    n, c, tail = 430000, 5120, 64
    x = torch.zeros(1, n, c, dtype=torch.bfloat16, device=cuda)
    g = torch.full((1, n, c), -0.25, dtype=torch.bfloat16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(1)
    x[:, -tail:] = torch.randn(1, tail, c, generator=gen, device=cuda).clamp(-5, 5).bfloat16()
    y, last = gated_scan(x, g)
    want, wlast = gated_scan(x[:, -tail:].contiguous(), g[:, -tail:].contiguous())
    assert not bool(y[:, :-tail].any())
    near = lambda a, b, fp32: bool(((a.float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + fp32).all())
    assert near(y[:, -tail:], want, 1e-4)
    assert float((last - wlast).abs().max()) < 1e-4
    grad = x
    grad[:, -tail:] = torch.randn(1, tail, c, generator=gen, device=cuda).clamp(-5, 5).bfloat16()
    y[:, -tail:] = want
    dx, dg, _ = gated_scan_backward(grad, g, y)
    wx, wg, _ = gated_scan_backward(grad[:, -tail:].contiguous(), g[:, -tail:].contiguous(), want)
    assert near(dx[:, -tail:], wx, 1e-4) and near(dg[:, -tail:], wg, 23e-4)


def test_steps_continue_a_scan(cuda):
    """Token by token with the state in place equals one call over all tokens."""
    from vdn_b200.recurrence import gated_scan
    gen, x, g = _case(8, (5, 12), 2, 64, torch.bfloat16, torch.float32, True)
    x, g = x.to(cuda), g.to(cuda)
    want, last = gated_scan(x, g)
    state = torch.zeros(5, 2, 64, device=cuda)
    ys = [gated_scan(x[:, t:t + 1], g[:, t:t + 1], state, out_state=state)[0] for t in range(12)]
    got = torch.cat(ys, 1)
    # the folds group the same sums differently: a few fp32 steps before the rounding to bf16
    assert float((state - last).abs().max()) <= 12 * 8 * U * float(last.abs().max() + x.float().abs().max()) * 12
    assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -8 * float(want.float().abs().max()) + 1e-6


def test_same_bits_every_run_and_on_other_streams(cuda):
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    gen, x, g = _case(9, (2, 3000), 4, 64, torch.bfloat16, torch.bfloat16, False)
    x, g = x.to(cuda), g.to(cuda)
    y, last = gated_scan(x, g)
    back = gated_scan_backward(x, g, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, last2 = gated_scan(x, g)
        back2 = gated_scan_backward(x, g, y2)
    y3, last3 = gated_scan(x, g)                         # meanwhile on this one
    torch.cuda.synchronize()
    assert torch.equal(y, y2) and torch.equal(y, y3) and torch.equal(last, last2) and torch.equal(last, last3)
    assert all(torch.equal(a, b) for a, b in zip(back, back2))


def test_gradients_against_differences(cuda):
    """d/dp of a weighted sum of outputs, by central differences in 64 bits of the reference."""
    from vdn_b200.recurrence import gated_scan
    gen, x, g = _case(2, (1, 40), 2, 32, torch.float32, torch.float32, True)
    s0 = torch.randn(1, 2, 32, generator=gen)
    wy, ws = torch.randn(40, 64, generator=gen).double(), torch.randn(64, generator=gen).double()

    def loss(xv, gv, sv):
        y, _, last = _scan(gv.repeat_interleave(32, 1).exp(), xv, sv)
        return (y * wy).sum() + (last * ws).sum()
    args = [x.to(cuda).requires_grad_(), g.to(cuda).requires_grad_(), s0.to(cuda).requires_grad_()]
    y, last = gated_scan(*args)
    ((y.flatten(2)[0] * wy.to(cuda).float()).sum() + (last.flatten() * ws.to(cuda).float()).sum()).backward()
    base = [x[0].flatten(1).double(), g[0].double(), s0.flatten().double()]
    for k, leaf in enumerate(args):
        direction = torch.randn(base[k].shape, generator=gen).double()
        plus, minus = ([b + sign * 1e-5 * direction if i == k else b for i, b in enumerate(base)] for sign in (1, -1))
        diff = (loss(*plus) - loss(*minus)) / 2e-5
        got = (leaf.grad.double().cpu().reshape(direction.shape) * direction).sum()
        scale = (leaf.grad.double().cpu().reshape(direction.shape) * direction).abs().sum()
        assert abs(float(got - diff)) < 1e-5 * float(scale), k   # 40 steps of fp32 and the difference's h^2


def test_capture_replay_and_refusal(cuda):
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    gen, x, g = _case(12, (2, 700), 2, 64, torch.bfloat16, torch.float32, False)
    x, g = x.to(cuda), g.to(cuda)
    want = gated_scan_backward(x, g, gated_scan(x, g)[0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    leaf = x.clone().requires_grad_()
    with torch.cuda.graph(graph):
        y, last = gated_scan(x, g)
        grads = gated_scan_backward(x, g, y)
        with pytest.raises(RuntimeError, match="capture"):
            gated_scan(leaf, g)
    x.mul_(2)
    graph.replay()
    again = gated_scan_backward(x, g, gated_scan(x, g)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    assert not torch.equal(grads[0], want[0])


def test_refusals(cuda):
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    x = torch.zeros(2, 4, 2, 32, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="log_decay"):
        gated_scan(x, x[:, :3])
    with pytest.raises(TypeError, match="log_decay"):
        gated_scan(x, x.half())
    with pytest.raises(ValueError, match="head dim"):
        gated_scan(x[..., :24], torch.zeros(2, 4, 2, dtype=torch.bfloat16, device=cuda))
    with pytest.raises(ValueError, match="cu_seqlens"):
        gated_scan(x[0], x[0], cu_seqlens=torch.zeros(3, dtype=torch.int64, device=cuda))
    with pytest.raises(ValueError, match="state"):
        gated_scan(x, x, torch.zeros(3, 2, 32, device=cuda))
    with pytest.raises(TypeError, match="state"):
        gated_scan(x, x, torch.zeros(2, 2, 32, device=cuda, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="out"):
        gated_scan(x, x, out=torch.zeros(2, 4, 2, 33, dtype=torch.bfloat16, device=cuda))
    with pytest.raises(ValueError, match="grad_y"):
        gated_scan_backward(x.float(), x, x)
    with pytest.raises(ValueError, match="recorded"):
        gated_scan(x.clone().requires_grad_(), x, out=torch.empty_like(x))


@pytest.mark.parametrize("shape", [(0, 5, 2, 32), (2, 0, 2, 32), (2, 5, 0, 32)])
def test_empty(cuda, shape):
    from vdn_b200.recurrence import gated_scan, gated_scan_backward
    x = torch.zeros(shape, dtype=torch.bfloat16, device=cuda)
    state = torch.ones(shape[0], *shape[2:], device=cuda)
    y, last = gated_scan(x, x, state)
    dx, dg, ds = gated_scan_backward(x, x, y, state=state, grad_state=2 * state)
    torch.cuda.synchronize()
    assert y.shape == dx.shape == dg.shape == x.shape
    if shape[1] == 0:
        assert torch.equal(last, state) and torch.equal(ds, 2 * state)
    none = gated_scan(x[0] if shape[0] else x.reshape(0, 2, 32), x[0] if shape[0] else x.reshape(0, 2, 32),
                      cu_seqlens=torch.zeros(1, dtype=torch.int32, device=cuda)) if shape[2] else None
    assert none is None or bool((none[0] == 0).all())
