"""The operators of a recurrent mixing layer: gated_scan, layer_norm and linear_act, forward and
backward, with the sizes that the framework's block (hidden 5120, 40 heads of 128, FFN 13824, 21
frames of 1560 tokens, 512 text rows) and its serving and training use give them."""
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
HIDDEN, HEADS, HEAD_DIM, FFN, ROWS, TEXT = 5120, 40, 128, 13824, 21 * 1560, 512


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of 64 requests, the state carried from call to call
        scan("scan_step_64", "forward", batch=64, tokens=1, heads=HEADS, dim=HEAD_DIM),
        # the whole clip as one sequence
        scan("scan_clip", "forward", batch=1, tokens=ROWS, heads=HEADS, dim=HEAD_DIM),
        # training: ragged clips packed into one row of tokens, one decay per head kept in 32 bits
        scan("scan_back_packed", "backward", batch=7, tokens=16389, heads=HEADS, dim=HEAD_DIM, packed=True, shared=True, decay="fp32"),
        # training in 32 bits, the reverse direction, an odd number of channels and tokens
        scan("scan_back_fp32", "backward", batch=3, tokens=1001, heads=1, dim=515, dtype="fp32", decay="fp32", reverse=True),
        # a norm in front of the block, whole clip
        norm("norm_clip", "forward", rows=ROWS, width=HIDDEN),
        # the norm of a decoding batch
        norm("norm_16", "forward", rows=16, width=HIDDEN, dtype="fp16"),
        # training: the norm's gradients over the whole clip, weights kept in 32 bits
        norm("norm_back_clip", "backward", rows=ROWS, width=HIDDEN, weight="fp32"),
        # training: per-head width, many short rows
        norm("norm_back_heads", "backward", rows=TEXT * HEADS + 1, width=HEAD_DIM),
        # FFN up for the tokens of a decoding batch: the weight's bytes are what it costs
        linear("linear_up_16", "forward", rows=16, n=FFN, k=HIDDEN, act="gelu_tanh"),
        # the output projection with the residual, whole clip
        linear("linear_out_clip", "forward", rows=ROWS, n=HIDDEN, k=HIDDEN, residual=True),
        # odd sizes, half precision, exact GELU, the text rows
        linear("linear_odd", "forward", rows=TEXT + 1, n=777, k=1004, act="gelu_erf", residual=True, dtype="fp16"),
        # training: FFN up over a quarter of the clip
        linear("linear_up_back", "backward", rows=ROWS // 4, n=FFN, k=HIDDEN, act="gelu_tanh"),
    ]


def scan(name, way, *, batch, tokens, heads, dim, dtype="bf16", decay="bf16", shared=False, packed=False, reverse=False, state=True):
    case = dict(op="scan", way=way, batch=batch, tokens=tokens, heads=heads, dim=dim, dtype=dtype, decay=decay, shared=shared,
                packed=packed, reverse=reverse, state=state)
    return dict(case, name=name) if name else case


def norm(name, way, *, rows, width, dtype="bf16", weight=None, bias=True):
    case = dict(op="norm", way=way, rows=rows, width=width, dtype=dtype, weight=weight or dtype, bias=bias)
    return dict(case, name=name) if name else case


def linear(name, way, *, rows, n, k, dtype="bf16", act="none", bias=True, residual=False):
    case = dict(op="linear", way=way, rows=rows, n=n, k=k, dtype=dtype, act=act, bias=bias, residual=residual)
    return dict(case, name=name) if name else case


def spread(rng, low, high):
    """A whole number, even over the logarithm."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op, way = rng.choice(["scan", "norm", "linear"]), rng.choice(["forward", "backward"])
    if op == "scan":
        shared = rng.random() < 0.4
        dim = rng.choice([32, 64, 128]) if shared else spread(rng, 8, 256)
        heads = spread(rng, 1, 48)
        tokens = spread(rng, 1, max(1, min(65536, ROWS * HIDDEN // (heads * dim))))
        packed = rng.random() < 0.4
        batch = spread(rng, 1, 64) if packed else spread(rng, 1, max(1, min(256, ROWS * HIDDEN // (heads * dim * tokens))))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return scan(None, way, batch=batch, tokens=tokens, heads=heads, dim=dim, dtype=dtype, decay=rng.choice([dtype, "fp32"]),
                    shared=shared, packed=packed, reverse=rng.random() < 0.5, state=rng.random() < 0.7)
    dtype = rng.choice(["bf16", "fp16"] if op == "linear" else ["bf16", "fp16", "fp32"])
    if op == "norm":
        width = spread(rng, 32, 16384)
        rows = spread(rng, 1, min(65536, ROWS * HIDDEN // width))
        if rng.random() < 0.6:
            width = -(-width // 64) * 64
        return norm(None, way, rows=rows, width=width, dtype=dtype, weight=rng.choice([dtype, "fp32"]), bias=rng.random() < 0.7)
    n, k = spread(rng, 64, FFN), spread(rng, 64, HIDDEN)
    if rng.random() < 0.7:
        n, k = -(-n // 64) * 64, -(-k // 64) * 64
    rows = spread(rng, 1, ROWS // 4)
    return linear(None, way, rows=rows, n=n, k=k, dtype=dtype, act=rng.choice(["none", "gelu_tanh", "gelu_erf", "silu"]),
                  bias=rng.random() < 0.7, residual=rng.random() < 0.5)


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    s = {"case": case}
    dtype = TYPES[case["dtype"]]
    if case["op"] == "scan":
        b, t, h, d = case["batch"], case["tokens"], case["heads"], case["dim"]
        lead = (t,) if case["packed"] else (b, t)
        rate = torch.rand(*lead, h, *([] if case["shared"] else [d]), generator=g, device=dev)
        # decays whose memory reaches from a token to some thousand tokens, as a trained gate's do
        s["log_decay"] = torch.exp(rate * 7.6 - 7.6).neg_().to(TYPES[case["decay"]])
        s["cu"] = None
        if case["packed"]:
            cuts = torch.randint(0, t + 1, (b - 1,), generator=g, device=dev, dtype=torch.int32).sort().values
            ends = torch.tensor([0, t], device=dev, dtype=torch.int32)
            s["cu"] = torch.cat([ends[:1], cuts, ends[1:]])
        s["state"] = normal(b, h, d) if case["state"] else None
        if case["way"] == "forward":
            s["x"] = normal(*lead, h, d, dtype=dtype)
        else:
            # what the forward pass left: its output, and the gradients that come back
            s["y"] = plain_scan(normal(*lead, h, d), s["log_decay"], s["state"], s["cu"], case["reverse"])[0].to(dtype)
            s["grad_y"] = normal(*lead, h, d, dtype=dtype)
            s["grad_state"] = normal(b, h, d) if case["state"] else None
    elif case["op"] == "norm":
        r, c = case["rows"], case["width"]
        s["x"] = (normal(r, c) * (0.5 + torch.rand(r, 1, generator=g, device=dev)) + normal(r, 1)).to(dtype)
        s["weight"] = (1 + 0.1 * normal(c)).to(TYPES[case["weight"]])
        s["bias"] = (0.1 * normal(c)).to(TYPES[case["weight"]]) if case["bias"] else None
        if case["way"] == "backward":
            s["grad_y"] = normal(r, c, dtype=dtype)
            x = s["x"].double()
            s["mean"] = x.mean(1).float()
            s["rstd"] = (x.var(1, unbiased=False) + 1e-5).rsqrt().float()
    else:
        r, n, k = case["rows"], case["n"], case["k"]
        s["x"] = normal(r, k, dtype=dtype)
        s["weight"] = (normal(n, k) * k ** -0.5).to(dtype)
        s["bias"] = (0.1 * normal(n)).to(dtype) if case["bias"] else None
        if case["way"] == "forward":
            s["residual"] = normal(r, n, dtype=dtype) if case["residual"] else None
        else:
            s["grad_y"] = normal(r, n, dtype=dtype)
            s["pre"] = None
            if case["act"] != "none":
                pre = s["x"].float() @ s["weight"].float().T
                s["pre"] = (pre if s["bias"] is None else pre + s["bias"].float()).to(dtype)
    return s


# --------------------------------------------------------------------------- one pass
def run(s):
    case = s["case"]
    if own:
        return run_own(case, s)
    dtype = TYPES[case["dtype"]]
    if case["op"] == "scan":
        if case["way"] == "forward":
            y, state = plain_scan(s["x"], s["log_decay"], s["state"], s["cu"], case["reverse"])
            return y.to(dtype), state
        dx, dg, ds = plain_scan_backward(s["grad_y"], s["log_decay"], s["y"], s["state"], s["grad_state"], s["cu"], case["reverse"])
        return (dx.to(dtype), dg.to(TYPES[case["decay"]])) + ((ds,) if case["state"] else ())
    if case["op"] == "norm":
        if case["way"] == "forward":
            x = s["x"].float()
            mean = x.mean(1, keepdim=True)
            xc = x - mean
            rstd = (xc.square().mean(1, keepdim=True) + 1e-5).rsqrt()
            y = xc * rstd * s["weight"].float()
            return (y if s["bias"] is None else y + s["bias"].float()).to(dtype)
        dy = s["grad_y"].float()
        xh = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
        wdy = dy * s["weight"].float()
        dx = (wdy - wdy.mean(1, keepdim=True) - xh * (wdy * xh).mean(1, keepdim=True)) * s["rstd"][:, None]
        kind = TYPES[case["weight"]]
        dw, db = (dy * xh).sum(0), dy.sum(0)
        return (dx.to(dtype), dw.to(kind)) + ((db.to(kind),) if case["bias"] else ())
    if case["way"] == "forward":
        z = s["x"].float() @ s["weight"].float().T
        y = act(z if s["bias"] is None else z + s["bias"].float(), case["act"])
        return (y if s["residual"] is None else y + s["residual"].float()).to(dtype)
    dz = s["grad_y"].float()
    if case["act"] != "none":
        dz = dz * act_slope(s["pre"].float(), case["act"])
    dx, dw, db = dz @ s["weight"].float(), dz.T @ s["x"].float(), dz.sum(0)
    return (dx.to(dtype), dw.to(dtype)) + ((db.to(dtype),) if case["bias"] else ())


def run_own(case, s):
    from vdn_b200.layer_norm import layer_norm, layer_norm_backward
    from vdn_b200.linear_act import linear_act, linear_act_backward
    from vdn_b200.recurrence import gated_scan, gated_scan_backward

    if case["op"] == "scan":
        more = dict(state=s["state"], cu_seqlens=s["cu"], reverse=case["reverse"])
        if case["way"] == "forward":
            return gated_scan(s["x"], s["log_decay"], **more)
        dx, dg, ds = gated_scan_backward(s["grad_y"], s["log_decay"], s["y"], grad_state=s["grad_state"], **more)
        return (dx, dg) + ((ds,) if case["state"] else ())
    if case["op"] == "norm":
        if case["way"] == "forward":
            return layer_norm(s["x"], s["weight"], s["bias"])
        grads = layer_norm_backward(s["grad_y"], s["x"], s["weight"], s["mean"], s["rstd"], bias=case["bias"])
    elif case["way"] == "forward":
        return linear_act(s["x"], s["weight"], s["bias"], act=case["act"], residual=s["residual"])
    else:
        grads = linear_act_backward(s["grad_y"], s["x"], s["weight"], s["pre"], act=case["act"], bias=case["bias"])
    return grads if case["bias"] else grads[:2]


# --------------------------------------------------------------------------- plain forms
def pieces(shape, cu):
    """First row and length of each sequence over rows laid end to end."""
    if cu is not None:
        return cu[:-1].long(), (cu[1:] - cu[:-1]).long()
    b, t = shape[:2]
    return torch.arange(b, device="cuda") * t, torch.full((b,), t, device="cuda")


def doubling(a, x):
    """h_t = a_t h_{t-1} + x_t over the rows, h_{-1} = 0, in log2(rows) steps that join neighbours."""
    step = 1
    while step < len(x):
        pad = (0, 0) * (x.dim() - 1) + (step, -step)
        x = x + a * torch.nn.functional.pad(x, pad)
        a = a * torch.nn.functional.pad(a, pad)
        step *= 2
    return x


def at_rows(rows, start, length, values):
    """[rows, ...] zeros with values[i] in row start[i], for the sequences that have a row."""
    place = torch.where(length > 0, start, rows)  # the others' go to a row behind the last
    return torch.zeros(rows + 1, *values.shape[1:], device="cuda").index_add_(0, place, values)[:rows]


def plain_scan(x, log_decay, state, cu, reverse):
    start, length = pieces(x.shape, cu)
    h, d = x.shape[-2:]
    rows = x.reshape(-1, h, d).float()
    a = log_decay.reshape(len(rows), h, -1).float().exp()
    n = len(rows)
    if reverse:
        rows, a, start = rows.flip(0), a.flip(0), n - start - length
    first = at_rows(n, start, length, torch.ones(len(start), 1, 1, device="cuda"))
    if state is not None:
        rows = rows + a * at_rows(n, start, length, state.float())
    y = doubling(a * (1 - first), rows)
    last = y[(start + length - 1).clamp(min=0)]
    old = torch.zeros_like(last) if state is None else state.float()
    final = torch.where((length > 0)[:, None, None], last, old)
    return (y.flip(0) if reverse else y).reshape(x.shape), final


def plain_scan_backward(grad_y, log_decay, y, state, grad_state, cu, reverse):
    start, length = pieces(y.shape, cu)
    h, d = y.shape[-2:]
    dy, y2 = grad_y.reshape(-1, h, d).float(), y.reshape(-1, h, d).float()
    n = len(dy)
    a = log_decay.reshape(n, h, -1).float().exp()
    if reverse:
        dy, y2, a, start = dy.flip(0), y2.flip(0), a.flip(0), n - start - length
    ones = torch.ones(len(start), 1, 1, device="cuda")
    first = at_rows(n, start, length, ones)
    last = at_rows(n, start + length - 1, length, ones)
    if grad_state is not None:
        dy = dy + at_rows(n, start + length - 1, length, grad_state.float())
    after = torch.nn.functional.pad(a[1:], (0, 0, 0, 0, 0, 1)) * (1 - last)
    u = doubling(after.flip(0), dy.flip(0)).flip(0)
    before = torch.nn.functional.pad(y2[:-1], (0, 0, 0, 0, 1, 0)) * (1 - first)
    if state is not None:
        before = before + at_rows(n, start, length, state.float())
    dg = a * u * before
    dg = dg.sum(2) if log_decay.dim() < y.dim() else dg
    into = (a * u)[start.clamp(max=n - 1)]
    back = torch.zeros_like(into) if grad_state is None else grad_state.float()
    ds = torch.where((length > 0)[:, None, None], into, back)
    if reverse:
        u, dg = u.flip(0), dg.flip(0)
    return u.reshape(y.shape), dg.reshape(log_decay.shape), ds


def act(z, kind):
    if kind == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3)))
    if kind == "gelu_erf":
        return 0.5 * z * (1 + torch.erf(z * 0.7071067811865476))
    return z * torch.sigmoid(z) if kind == "silu" else z


def act_slope(z, kind):
    if kind == "gelu_tanh":
        t = torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * 0.7978845608028654 * (1 + 0.134145 * z * z)
    if kind == "gelu_erf":
        return 0.5 * (1 + torch.erf(z * 0.7071067811865476)) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    p = torch.sigmoid(z)
    return p * (1 + z * (1 - p))


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = SIZE[case["dtype"]]
    back = case["way"] == "backward"
    if case["op"] == "scan":
        rows = case["tokens"] * (1 if case["packed"] else case["batch"])
        full, few = rows * case["heads"] * case["dim"], rows * case["heads"]
        decays = (few if case["shared"] else full) * SIZE[case["decay"]]
        states = case["batch"] * case["heads"] * case["dim"] * 4
        if back:
            return {"bytes": 3 * full * e + 2 * decays + (3 * states if case["state"] else 0), "flops": 5 * full}
        return {"bytes": 2 * full * e + decays + (2 if case["state"] else 1) * states, "flops": 2 * full}
    if case["op"] == "norm":
        full, w = case["rows"] * case["width"], case["width"] * SIZE[case["weight"]] * (2 if case["bias"] else 1)
        if back:
            return {"bytes": 3 * full * e + 8 * case["rows"] + w + case["width"] * SIZE[case["weight"]], "flops": 13 * full}
        return {"bytes": 2 * full * e + w, "flops": 8 * full}
    r, n, k = case["rows"], case["n"], case["k"]
    if back:
        pre = r * n if case["act"] != "none" else 0
        return {"bytes": e * (r * n + pre + 2 * r * k + 2 * n * k + (n if case["bias"] else 0)), "flops": 4 * r * n * k}
    return {"bytes": e * (r * k + n * k + r * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)), "flops": 2 * r * n * k}


# --------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if case["op"] == "scan":
        return exact_scan(case, wide)
    if case["op"] == "norm":
        x, w = wide["x"], wide["weight"].expand(case["rows"], -1)
        if case["way"] == "forward":
            var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
            y = w * (x - mean) / torch.sqrt(var + 1e-5)
            return y if s["bias"] is None else y + wide["bias"]
        dy, mean, rstd = wide["grad_y"], wide["mean"].unsqueeze(1), wide["rstd"].unsqueeze(1)
        dxh, xh, c = dy * w, (x - mean) * rstd, case["width"]
        dx = rstd / c * (c * dxh - dxh.sum(1, keepdim=True) - xh * torch.einsum("rc,rc->r", dxh, xh).unsqueeze(1))
        return (dx, torch.einsum("rc,rc->c", dy, xh)) + ((torch.einsum("rc->c", dy),) if case["bias"] else ())
    z = wide["pre"] if case["way"] == "backward" and case["act"] != "none" else None
    if case["way"] == "forward":
        z = torch.nn.functional.linear(wide["x"], wide["weight"], wide["bias"])
    value, slope = exact_act(z, case["act"]) if z is not None else (None, None)
    if case["way"] == "forward":
        return value if s["residual"] is None else wide["residual"] + value
    dz = wide["grad_y"] if slope is None else wide["grad_y"] * slope
    grads = (torch.mm(dz, wide["weight"]), torch.mm(dz.t(), wide["x"]))
    return grads + ((torch.mv(dz.t(), torch.ones_like(dz[:, 0])),) if case["bias"] else ())


def exact_act(z, kind):
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "gelu_erf":
        cdf = 0.5 * torch.erfc(-z / 2.0 ** 0.5)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
    if kind == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p + z * p * (1 - p)
    root = (2 / torch.pi) ** 0.5
    p = 1 / (1 + torch.exp(-2 * root * (z + 0.044715 * z ** 3)))  # 0.5 (1 + tanh u) = sigmoid(2 u)
    return z * p, p + 2 * root * z * p * (1 - p) * (1 + 3 * 0.044715 * z * z)


def exact_scan(case, s):
    b, h, d = case["batch"], case["heads"], case["dim"]
    decay = torch.exp(s["log_decay"].unsqueeze(-1) if case["shared"] else s["log_decay"])
    forward = case["way"] == "forward"
    main = s["x"] if forward else s["grad_y"]
    if case["packed"]:
        cu = s["cu"].tolist()
        spans = [(i, slice(lo, hi)) for i, (lo, hi) in enumerate(zip(cu, cu[1:]))]
    else:
        spans = [(slice(None), None)]  # all sequences side by side, token by token
    zeros = torch.zeros(b, h, d, dtype=torch.float64, device="cuda")
    first = zeros if s["state"] is None else s["state"]
    out, dg = torch.zeros_like(main), torch.zeros_like(main)
    last = zeros.clone()
    for i, span in spans:
        def part(v):
            return v[span] if span is not None else v.transpose(0, 1)  # [tokens, ...]
        m, a, o = part(main), part(decay), part(out)
        order = range(len(m) - 1, -1, -1) if case["reverse"] else range(len(m))
        if forward:
            hold = first[i]
            for t in order:
                hold = torch.addcmul(m[t], a[t], hold)
                o[t] = hold
        else:
            y, g = part(s["y"]), part(dg)
            hold = zeros[i] if s["grad_state"] is None else s["grad_state"][i]
            order = list(order)
            for at in range(len(order) - 1, -1, -1):
                t = order[at]
                o[t] = m[t] + hold
                hold = a[t] * o[t]
                g[t] = hold * (y[order[at - 1]] if at else first[i])
        last[i] = hold
    if forward:
        return out, last
    return (out, dg.sum(-1) if case["shared"] else dg) + ((last,) if case["state"] else ())
