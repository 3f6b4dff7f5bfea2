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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width,shared", [(128, False), (65, False), (128, True)])   # tensor maps, plain loads, heads
@pytest.mark.parametrize("cu", [None, [3, 40, 40, 900, 1200]])
def test_in_place_outputs(cuda, dtype, width, shared, cu):
    """out over x or log_decay gives the bits of a call with memory of its own."""
    from vdn_b200.recurrence import gated_scan
    gen = torch.Generator().manual_seed(2)
    lead = (1300,) if cu else (2, 700)
    tail = (2, 64) if shared else (width,)
    x = torch.randn(*lead, *tail, generator=gen).to(dtype).to(cuda)
    g = (-torch.rand(*lead, *tail[:1], generator=gen)).to(dtype).to(cuda)
    cud = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=cuda)
    state = torch.randn(len(cu) - 1 if cu else 2, *tail, generator=gen).to(cuda)
    inside = slice(None) if cu is None else slice(cu[0], cu[-1])
    want, last = gated_scan(x, g, state, cu_seqlens=cud)
    for over in ("x", "log_decay"):
        if shared and over == "log_decay":
            continue
        a, b, s = x.clone(), g.clone(), state.clone()
        y, end = gated_scan(a, b, s, cu_seqlens=cud, out=a if over == "x" else b, out_state=s)
        assert y is (a if over == "x" else b) and end is s
        assert torch.equal(y[inside], want[inside]) and torch.equal(end, last)


def test_columns_of_one_buffer(cuda):
    """Rows that lie side by side in one buffer share no memory, whatever their addresses' ranges."""
    from vdn_b200.recurrence import gated_scan
    x, g, state = _args(cuda, 40)
    want = gated_scan(x, g, state)
    buffer = torch.zeros(2, 40, 5 * 128, device=cuda)
    part = [buffer[..., i * 128:(i + 1) * 128].unflatten(-1, (2, 64)) for i in range(5)]
    part[0].copy_(x)
    part[2].copy_(g)
    y, last = gated_scan(part[0], part[2], state, out=part[3])
    assert torch.equal(y, want[0]) and torch.equal(last, want[1])
    turned = buffer.transpose(0, 1).contiguous().transpose(0, 1)       # token-major
    part = [turned[..., i * 128:(i + 1) * 128].unflatten(-1, (2, 64)) for i in range(5)]
    assert torch.equal(gated_scan(part[0], part[2], state, out=part[4])[0], want[0])
    for buffer in (torch.zeros(4, 40, 2, 64, device=cuda), torch.zeros(2, 80, 2, 64, device=cuda)):
        part = [buffer[i::2] if len(buffer) == 4 else buffer[:, i::2] for i in range(2)]    # every other batch, every other row
        part[1].copy_(x)
        assert torch.equal(gated_scan(part[1], g, state, out=part[0])[0], want[0])
    one = [t[:, :1] for t in (x, g)]                                   # a step keeps its state in its output
    want = gated_scan(*one, state)
    hold = state.clone()
    gated_scan(*one, hold, out=hold[:, None], out_state=hold)
    assert torch.equal(hold, want[1])


def test_shared_memory_is_refused(cuda):
    from vdn_b200.recurrence import gated_scan
    x, g, state = _args(cuda, 40)
    buffer = torch.zeros(2 * 41 * 128 + 128, device=cuda)
    first, second = (buffer[o:o + x.numel()].view(x.shape) for o in (0, 128))     # a row apart
    with pytest.raises(ValueError, match="same rows"):
        gated_scan(first, g, state, out=second)
    with pytest.raises(ValueError, match="same rows"):
        gated_scan(x, second, state, out=first)
    with pytest.raises(ValueError, match="overlap"):
        gated_scan(x, g, state, out=torch.empty_like(x[:, :1]).expand(x.shape))
    with pytest.raises(ValueError, match="overlap"):
        gated_scan(x, g, state, out=torch.empty(2, 40 * 64 + 128, device=cuda).as_strided(x.shape, (40 * 64 + 128, 64, 64, 1)))
    wide = torch.zeros(2, 40, 300, device=cuda)
    with pytest.raises(ValueError, match="same rows"):                            # columns that overlap
        gated_scan(wide[..., :128].unflatten(-1, (2, 64)), g, state, out=wide[..., 100:228].unflatten(-1, (2, 64)))
    pool = torch.zeros(3, 2, 64, device=cuda)
    with pytest.raises(ValueError, match="out_state and state"):
        gated_scan(x, g, pool[:2], out_state=pool[1:])
    with pytest.raises(ValueError, match="out and state"):
        gated_scan(x, g, x.view(-1)[:256].view(2, 2, 64), out=x)
    with pytest.raises(ValueError, match="out and out_state"):
        out = torch.empty_like(x)
        gated_scan(x, g, state, out=out, out_state=out.view(-1)[:256].view(2, 2, 64))
    with pytest.raises(ValueError, match="out_state and x"):
        gated_scan(x, g, state, out_state=x.view(-1)[:256].view(2, 2, 64))
    with pytest.raises(ValueError, match="out_state and log_decay"):
        gated_scan(x, g, state, out_state=g.view(-1)[:256].view(2, 2, 64))
