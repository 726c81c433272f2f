"""The operators of row-normalised residual blocks and of their weights' update, as measurable cases.

Two families, each in its plain form (elementary torch operations in 32 bits) and through the framework's entry points:

  row norms   ``norm_ops.row_norm_act``: y = act(norm(x)), the norm before a block; ``norm_ops.row_norm_join``:
              y = act(r + keep[b] gate[b] scale norm(z)), optionally with h = norm(y) of the next block: the norm after a block
              fused with its gate (per plot and channel), drop-path factor, per-channel residual scale, shortcut, activation
  updates     ``muon_ops.orthogonalize``: five Newton-Schulz iterations x <- a x + (b g + c g g) x, g = x x^T, of a stack of
              matrices; ``muon_ops.muon_update``: momentum, orthogonalisation, weight decay and step of a list of parameters
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MOMENTUM, LR, DECAY, NORM_EPS, ORTHO_EPS = 0.95, 0.005, 0.01, 1e-6, 1e-7
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _senet14():
    """(rows, cols) of the weight matrices of the SENet14 backbone: kernels [offsets * Cin, Cout], shortcuts, excitations."""
    shapes, cin = [(343 * 3, 64)], 64
    for cout in (64, 128, 256, 512):
        shapes += [(27 * cin, cout), (27 * cout, cout), (cout // 16, cout), (cout, cout // 16)]
        if cin != cout:
            shapes.append((cin, cout))
        cin = cout
    return ",".join("%dx%d" % s for s in shapes)


def listed():
    norm = dict(op="norm", plots=32, kind="layer", act="gelu", gate=True, keep=True, scale=True, next=False)
    ortho = dict(op="ortho", batch=1, dtype="fp32")
    return [
        # one pooled row for each plot of a batch, in front of the regression head, at inference: latency
        dict(norm, name="norm-serve-32x512", form="act", rows=32, cols=512, dtype="fp32", train=False, act="none"),
        # the first level of the sparse backbone (32 plots), fp32 rows: norm and activation behind its convolution
        dict(norm, name="norm-act-train-211000x64", form="act", rows=211000, cols=64, dtype="fp32", train=True),
        # root-mean-square norm of a wide bottleneck level on bf16 rows
        dict(norm, name="norm-act-train-61007x512-rms", form="act", rows=61007, cols=512, dtype="bf16", train=True, kind="rms",
             act="relu"),
        # the join of one plot's bottleneck block at inference
        dict(norm, name="join-serve-1901x1024", form="join", rows=1901, cols=1024, plots=1, dtype="bf16", train=False, keep=False),
        # the widest level of the 50-layer backbone on bf16 rows: block tail, forward and backward; the largest of the norms
        dict(norm, name="join-train-211000x256", form="join", rows=211000, cols=256, dtype="bf16", train=True),
        # odd widths, fp32, with the norm of the next block behind the join
        dict(norm, name="join-next-train-50021x203", form="join", rows=50021, cols=203, dtype="fp32", train=True, kind="rms",
             act="none", next=True),
        # one small linear layer: latency
        dict(ortho, name="ortho-64x64", rows=64, cols=64),
        # a convolution kernel taken one offset at a time
        dict(ortho, name="ortho-27x128x128-bf16", batch=27, rows=128, cols=128, dtype="bf16"),
        # odd sizes
        dict(ortho, name="ortho-3x515x1029", batch=3, rows=515, cols=1029),
        # the largest convolution kernel of the backbone as one matrix
        dict(ortho, name="ortho-13824x512", rows=13824, cols=512),
        # a large square matrix: the largest of the updates
        dict(ortho, name="ortho-2048x2048-bf16", rows=2048, cols=2048, dtype="bf16"),
        # the whole update of the backbone's weight matrices, as every training step makes it
        dict(op="update", name="update-senet14", shapes=_senet14(), nesterov=True),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "ortho", "ortho", "update"])
    if op == "norm":
        cols = _between(rng, 4, 2048)
        rows = _between(rng, 1, max(2, min(211000, 211000 * 256 // cols)))
        form = rng.choice(["act", "join"])
        return dict(op=op, form=form, rows=rows, cols=cols, plots=rng.randint(1, 64), dtype=rng.choice(["fp32", "bf16"]),
                    train=rng.random() < 0.7, kind=rng.choice(["layer", "rms"]), act=rng.choice(["none", "relu", "gelu"]),
                    gate=rng.random() < 0.7, keep=rng.random() < 0.7, scale=rng.random() < 0.7,
                    next=form == "join" and rng.random() < 0.4)
    if op == "ortho":
        short = _between(rng, 2, 1536)
        long = _between(rng, short, max(short + 1, min(13824, 3 * 10 ** 6 // short)))
        room = max(1, min(64, 2 * 10 ** 9 // (short * short * long)))
        rows, cols = rng.choice([(short, long), (long, short)])
        return dict(op=op, batch=_between(rng, 1, room), rows=rows, cols=cols, dtype=rng.choice(["fp32", "bf16", "fp16"]))
    shapes = []
    for _ in range(rng.randint(1, 12)):
        short = _between(rng, 2, 512)
        long = _between(rng, short, 27 * short)
        shapes.append("%dx%d" % rng.choice([(short, long), (long, short)]))
    return dict(op=op, shapes=",".join(shapes), nesterov=rng.random() < 0.7)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _gradient(gen, dev, batch, rows, cols):
    """Gradients of linear layers, inputs^T errors: rectified inputs (one strong direction: their mean), errors of unequal
    size."""
    n = max(rows, cols) + 32
    inputs = torch.relu(torch.randn(batch, n, min(rows, cols), device=dev, generator=gen))
    errors = torch.randn(batch, n, max(rows, cols), device=dev, generator=gen)
    errors *= torch.exp(0.5 * torch.randn(batch, 1, max(rows, cols), device=dev, generator=gen)) * 1e-3
    g = torch.matmul(inputs.transpose(1, 2).contiguous(), errors)
    return g if rows <= cols else g.transpose(1, 2).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "ortho":
        s["x"] = _gradient(gen, dev, case["batch"], case["rows"], case["cols"]).to(DTYPES[case["dtype"]])
        return s
    if case["op"] == "update":
        shapes = _shapes(case)
        s["grads"] = [_gradient(gen, dev, 1, r, c)[0] for r, c in shapes]
        s["momenta"] = [0.3 * _gradient(gen, dev, 1, r, c)[0] for r, c in shapes]
        s["params"] = [0.02 * torch.randn(r, c, device=dev, generator=gen) for r, c in shapes]
        return s
    n, c, b = case["rows"], case["cols"], case["plots"]
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    def rows():       # channels of unequal spread and mean, as a convolution leaves them
        return (randn(n, c) * torch.exp(0.3 * randn(1, c)) + 0.5 * randn(1, c)).to(dt)

    s["z"], s["w"], s["bias"] = rows(), 1 + 0.1 * randn(c), (0.1 * randn(c) if case["kind"] == "layer" else None)
    if case["form"] == "join":
        # plots of unequal length, rows in plot order; a plot may be empty
        share = torch.rand(b, device=dev, generator=gen) ** 2
        share[torch.randint(b, (1,), device=dev, generator=gen)] += 1.0
        ptr = torch.cat([torch.zeros(1, device=dev), torch.cumsum(share, 0) / share.sum()])
        ptr = (ptr * n).round().to(torch.int32)
        ptr[-1] = n
        s["r"], s["ptr"] = rows(), ptr
        s["plot"] = torch.bucketize(torch.arange(n, device=dev, dtype=torch.int32), ptr[1:].contiguous(), right=True)
        s["gate"] = torch.sigmoid(randn(b, c)) if case["gate"] else None
        s["keep"] = (torch.rand(b, device=dev, generator=gen) > 0.1).float() / 0.9 if case["keep"] else None
        s["scale"] = 0.1 + 0.02 * randn(c) if case["scale"] else None
        s["w2"] = 1 + 0.1 * randn(c) if case["next"] else None
        s["dh"] = randn(n, c).to(dt) if case["next"] else None
    s["dy"] = randn(n, c).to(dt) if case["train"] else None
    for k in ("z", "r", "w", "bias", "gate", "scale", "w2"):      # the leaves of a training step
        if case["train"] and s.get(k) is not None:
            s[k].requires_grad_()
    return s


LEAVES = ("z", "r", "w", "bias", "gate", "scale", "w2")


def _leaves(s):
    return [k for k in LEAVES if s.get(k) is not None]


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_norm(x, w, bias, kind):
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    y = x / torch.sqrt((x * x).mean(1, keepdim=True) + NORM_EPS) * w
    return y if bias is None else y + bias


def _plain_act(u, act):
    if act == "relu":
        return torch.clamp(u, min=0)
    if act == "gelu":
        return 0.5 * u * (1 + torch.erf(u * math.sqrt(0.5)))
    return u


def _plain_forward(s):
    case = s["case"]
    y = _plain_norm(s["z"].float(), s["w"], s["bias"], case["kind"])
    if case["form"] == "act":
        return _plain_act(y, case["act"]).to(s["z"].dtype), None
    if s["scale"] is not None:
        y = y * s["scale"]
    if s["keep"] is not None or s["gate"] is not None:
        f = s["gate"] if s["keep"] is None else s["keep"][:, None] if s["gate"] is None else s["gate"] * s["keep"][:, None]
        y = y * f.index_select(0, s["plot"])
    y = _plain_act(y + s["r"].float(), case["act"])
    h = _plain_norm(y, s["w2"], None, case["kind"]).to(s["z"].dtype) if case["next"] else None
    return y.to(s["z"].dtype), h


def _plain_orthogonalize(x):
    x = x.float()
    wide = x.shape[1] <= x.shape[2]
    x = x if wide else x.transpose(1, 2)
    norm = torch.sqrt(torch.sum(x.double() ** 2, dim=(1, 2), keepdim=True)) + ORTHO_EPS
    x = (x / norm).float()
    a, b, c = COEFFICIENTS
    for _ in range(5):
        g = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
    return x if wide else x.transpose(1, 2)


def _plain_update(p, g, m, nesterov):
    m.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
    u = g * (1 - MOMENTUM) + m * MOMENTUM if nesterov else m
    o = _plain_orthogonalize(u[None])[0]
    p.mul_(1 - LR * DECAY).add_(o, alpha=-LR * 0.2 * math.sqrt(max(p.shape)))


# ------------------------------------------------------------------------------------------------ one pass
def _own_forward(s):
    from dpcr_agb_amd import norm_ops
    case = s["case"]
    if case["form"] == "act":
        return norm_ops.row_norm_act(s["z"], s["w"], s["bias"], NORM_EPS, case["kind"], case["act"]), None
    out = norm_ops.row_norm_join(s["z"], s["r"], s["w"], s["bias"], NORM_EPS, case["kind"], case["act"], gate=s["gate"],
                                 keep=s["keep"], ptr=s["ptr"], scale=s["scale"],
                                 next_norm=(s["w2"], None) if case["next"] else None)
    return out if case["next"] else (out, None)


def run(s):
    case = s["case"]
    if case["op"] == "ortho":
        if own:
            from dpcr_agb_amd import muon_ops
            return muon_ops.orthogonalize(s["x"], 5, COEFFICIENTS, ORTHO_EPS)
        return _plain_orthogonalize(s["x"]).to(s["x"].dtype).contiguous()
    if case["op"] == "update":
        if own:
            from dpcr_agb_amd import muon_ops
            muon_ops.muon_update(s["params"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM, nesterov=case["nesterov"],
                                 weight_decay=DECAY, steps=5, coefficients=COEFFICIENTS, eps=ORTHO_EPS, adjust="rms")
        else:
            for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
                _plain_update(p, g, m, case["nesterov"])
        return {"params": s["params"], "momenta": s["momenta"]}
    y, h = (_own_forward if own else _plain_forward)(s)
    if not case["train"]:
        return {"y": y, "h": h}
    keys = _leaves(s)
    outs, douts = ([y], [s["dy"]]) if h is None else ([y, h], [s["dy"], s["dh"]])
    grads = torch.autograd.grad(outs, [s[k] for k in keys], douts)
    return {"y": y.detach(), "h": None if h is None else h.detach(), **{"d" + k: g for k, g in zip(keys, grads)}}


def work(case):
    if case["op"] == "norm":
        e, n = (4 if case["dtype"] == "fp32" else 2), case["rows"] * case["cols"]
        join, nxt = case["form"] == "join", case["next"]
        tensors = 2 + join + nxt                                   # z (r) in, y (h) out
        if case["train"]:
            tensors += 2 + 2 * join + nxt                          # dy (dh) in and dz (dr) out; z and r are read once
        return {"bytes": tensors * n * e, "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "ortho":
        shapes, e, extra = [(case["rows"], case["cols"])] * case["batch"], 4 if case["dtype"] == "fp32" else 2, 0
    else:
        shapes, e, extra = _shapes(case), 4, 3                     # parameter, momentum in and out, gradient in
    flops = elems = 0
    for r, c in shapes:
        k, n = min(r, c), max(r, c)
        # g and g g are symmetric: half their products; x' = x + B x
        flops += 5 * (k * k * n + k ** 3 + 2 * k * k * n)
        elems += r * c
    return {"bytes": elems * e * (2 + extra), "flops": flops}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_normed(x, kind):
    if kind == "layer":
        x = x - x.sum(1, keepdim=True) / x.shape[1]
    rstd = (x.square().sum(1, keepdim=True) / x.shape[1] + NORM_EPS).rsqrt()
    return x * rstd, rstd


def _exact_norm_grad(dxhat, xhat, rstd, kind):
    """dL/dx from dL/dxhat: its part along xhat (and, for a centred norm, along the ones) is removed."""
    d = dxhat - xhat * (dxhat * xhat).mean(1, keepdim=True)
    if kind == "layer":
        d = d - dxhat.mean(1, keepdim=True)
    return d * rstd


def _exact_norm(case, s):
    kind, join = case["kind"], case["form"] == "join"
    d = {k: (v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in s.items()}
    n, c = d["z"].shape
    zhat, rstd = _exact_normed(d["z"], kind)
    bias = d["bias"] if d["bias"] is not None else torch.zeros_like(d["w"])
    norm = zhat * d["w"] + bias
    if join:
        scale = d["scale"] if d["scale"] is not None else torch.ones_like(d["w"])
        gate = d["gate"] if d["gate"] is not None else torch.ones(case["plots"], c, device=norm.device, dtype=torch.float64)
        keep = d["keep"] if d["keep"] is not None else torch.ones(case["plots"], device=norm.device, dtype=torch.float64)
        factor = (gate * keep[:, None] * scale)[d["plot"]]
        u = d["r"] + factor * norm
    else:
        u = norm
    if case["act"] == "relu":
        y, slope = u * (u > 0), (u > 0).double()
    elif case["act"] == "gelu":
        phi = torch.special.ndtr(u)
        y, slope = u * phi, phi + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)
    else:
        y, slope = u, torch.ones_like(u)
    out = {"y": y, "h": None}
    if case["next"]:
        yhat, rstd2 = _exact_normed(y, kind)
        out["h"] = yhat * d["w2"]
    if not case["train"]:
        return out
    dy = d["dy"]
    if case["next"]:
        out["dw2"] = (d["dh"] * yhat).sum(0)
        dy = dy + _exact_norm_grad(d["dh"] * d["w2"], yhat, rstd2, kind)
    du = dy * slope
    dnorm = du
    if join:
        out["dr"] = du
        dnorm = du * factor
        per_plot = torch.zeros(case["plots"], c, device=du.device, dtype=torch.float64)
        per_plot.index_add_(0, d["plot"].long(), du * norm)
        if d["gate"] is not None:
            out["dgate"] = per_plot * keep[:, None] * scale
        if d["scale"] is not None:
            out["dscale"] = (per_plot * gate * keep[:, None]).sum(0)
    out["dz"] = _exact_norm_grad(dnorm * d["w"], zhat, rstd, kind)
    out["dw"] = (dnorm * zhat).sum(0)
    if d["bias"] is not None:
        out["dbias"] = dnorm.sum(0)
    return out


def _exact_orthogonalize(x):
    """The same polynomial of every singular value, through x^T x of the shorter side: x p(x^T x) step by step."""
    tall = x.shape[-2] >= x.shape[-1]
    x = x if tall else x.mT
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + ORTHO_EPS)
    a, b, c = COEFFICIENTS
    eye = torch.eye(x.shape[-1], device=x.device, dtype=x.dtype)
    for _ in range(5):
        g = x.mT.contiguous() @ x
        x = x @ (a * eye + g @ (b * eye + c * g))
    return (x if tall else x.mT).contiguous()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(case, s)
    if case["op"] == "ortho":
        return _exact_orthogonalize(s["x"].double())
    params, momenta = [], []
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        g, m = g.double(), m.double() * MOMENTUM + g.double() * (1 - MOMENTUM)
        u = m * MOMENTUM + g * (1 - MOMENTUM) if case["nesterov"] else m
        step = LR * 0.2 * math.sqrt(max(p.shape))
        params.append(p.double() * (1 - LR * DECAY) - step * _exact_orthogonalize(u))
        momenta.append(m)
    return {"params": params, "momenta": momenta}
