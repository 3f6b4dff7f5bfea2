"""GPU: norm, projections, gated scan and output projection run together as a recurrent mixing
layer does, forward and backward, trained by autograd and served token by token.

    h = layer_norm(x);  v = silu(h Wv^T + bv);  g = -softplus(h Wg^T + bg)
    s = gated_scan(v, g);  y = x + s Wo^T + bo

The reference is the same composition in 64 bits on the same 16-bit parameters and input.
Each of the seven values handed on (h, v, the decay's projection and its softplus, s, y, and
in the backward their gradients) is rounded to 16 bits, 2^-8 of itself at most; a gradient passes through
about twelve such roundings, each of which a matrix product averages.  The 2-norm of the
error is held to 12 * 2^-8 / sqrt(3) (evenly spread rounding errors) of the 2-norm."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

B, T, H, D = 2, 150, 4, 64
C = H * D
LIMIT = 12 * 2.0 ** -8 / 3 ** 0.5


def _parameters():
    gen = torch.Generator().manual_seed(0)

    def matrix():
        return (torch.randn(C, C, generator=gen) * C ** -0.5).bfloat16()
    return dict(nw=(1 + 0.1 * torch.randn(C, generator=gen)).bfloat16(), nb=(0.1 * torch.randn(C, generator=gen)).bfloat16(),
                wv=matrix(), bv=(0.1 * torch.randn(C, generator=gen)).bfloat16(), wg=matrix(),
                bg=(torch.randn(C, generator=gen) - 2).bfloat16(), wo=matrix(), bo=(0.1 * torch.randn(C, generator=gen)).bfloat16(),
                x=torch.randn(B, T, C, generator=gen).bfloat16()), torch.randn(B, T, C, generator=gen).bfloat16()


def _layer(p, x, state=None):
    from vdn_b200.layer_norm import layer_norm
    from vdn_b200.linear_act import linear_act
    from vdn_b200.recurrence import gated_scan
    h = layer_norm(x, p["nw"], p["nb"])
    v = linear_act(h, p["wv"], p["bv"], act="silu")
    g = -F.softplus(linear_act(h, p["wg"], p["bg"]).float()).to(x.dtype)
    shape = (*x.shape[:2], H, D)
    s, last = gated_scan(v.view(shape), g.view(shape), state)
    return linear_act(s.flatten(2), p["wo"], p["bo"], residual=x), last


def _reference(p, x):
    h = F.layer_norm(x, (C,), p["nw"], p["nb"])
    v = F.silu(h @ p["wv"].T + p["bv"])
    a = torch.exp(-F.softplus(h @ p["wg"].T + p["bg"]))
    state, out = torch.zeros_like(x[:, 0]), []
    for t in range(x.shape[1]):
        state = a[:, t] * state + v[:, t]
        out.append(state)
    return x + torch.stack(out, 1) @ p["wo"].T + p["bo"], state


def _far(got, want):
    return float((got.double().cpu() - want).norm() / want.norm())


def test_training_step(cuda):
    params, dy = _parameters()
    leaves = {k: t.to(cuda).requires_grad_() for k, t in params.items()}
    y, last = _layer(leaves, leaves["x"])
    y.backward(dy.to(cuda))
    wide = {k: t.double().requires_grad_() for k, t in params.items()}
    ref, ref_last = _reference(wide, wide["x"])
    ref.backward(dy.double())
    assert _far(y.detach(), ref.detach()) < LIMIT
    assert _far(last.detach().flatten(1), ref_last.detach()) < LIMIT
    for k in params:
        assert leaves[k].grad.dtype == torch.bfloat16
        assert _far(leaves[k].grad, wide[k].grad) < LIMIT, k


@torch.no_grad()
def test_serving_token_by_token(cuda):
    """A prompt in one call, then single tokens that carry the state, against one call over all."""
    params, _ = _parameters()
    p = {k: t.to(cuda) for k, t in params.items()}
    whole, last = _layer(p, p["x"])
    y, state = _layer(p, p["x"][:, :100])
    parts = [y]
    for t in range(100, T):
        y, state = _layer(p, p["x"][:, t:t + 1], state)
        parts.append(y)
    assert _far(torch.cat(parts, 1), whole.double().cpu()) < LIMIT
    assert _far(state, last.double().cpu()) < LIMIT


@torch.no_grad()
def test_step_in_a_graph(cuda):
    """The serving step captured once and replayed for every token."""
    params, _ = _parameters()
    p = {k: t.to(cuda) for k, t in params.items()}
    state = torch.zeros(B, H, D, device=cuda)
    token = p["x"][:, :1].clone()

    def step():
        y, new = _layer(p, token, state)
        state.copy_(new)
        return y
    eager = []
    for t in range(20):
        token.copy_(p["x"][:, t:t + 1])
        eager.append(step().clone())
    state.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    state.zero_()
    for t in range(20):
        token.copy_(p["x"][:, t:t + 1])
        graph.replay()
        assert torch.equal(out, eager[t]), t
