"""Timed operators around the mixture-of-experts layer: what a training step does beside the layer's own products.

* ``join`` / ``join_backward`` — a sub-layer's output joined to the residual stream: a norm behind the sub-layer, a gate, a
  residual scale, the add, and the norm in front of the next sub-layer, in one call each way (``ResidualJoin``);
* ``orthogonalize`` — Newton-Schulz products that bring every singular value of a matrix near one (``Muon``);
* ``muon`` — the optimiser step around it: momentum, orthogonalised update, decoupled decay, for a stack of weights.

Sizes are those of the layers in ``rustingbrain_amd.synth.WORKLOADS`` and of the default ``TransformerConfig``: rows of 512 to
1024 (drawn ones up to 2048 and off every tile), calls of 1 to 16384 rows, experts of 352 to 1408, 8 to 64 a layer.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
# coefficients of the quintic a x + b x^3 + c x^5 whose iterates bring [0.003, 1] to about [0.68, 1.21] in five steps
NS = (3.4445, -4.7750, 2.0315)

_TORCH = {"bf16": torch.bfloat16, "f32": torch.float32}


def _join(kind, rows, cols, dtype, gate, post=True, following=True, padding=0.0, **more):
    return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, gate=gate, post=post, following=following, padding=padding, **more)


def _matrices(kind, count, rows, cols, dtype, **more):
    return dict(kind=kind, count=count, rows=rows, cols=cols, dtype=dtype, **more)


def listed():
    return [
        # one token of one conversation through the default model, norms on both sides and a gate a channel: all latency
        _join("join", 1, 512, "bf16", "channel", name="join_one_row"),
        # a serving step of decode rows and short prompts, padded to the batch; the residual scale alone, no norm behind
        _join("join", 203, 768, "bf16", "none", post=False, padding=0.1, name="join_serving_mixed"),
        # three sequences in the reference's own precision, a width that no vector divides, gated by token
        _join("join", 1533, 1365, "f32", "row", name="join_f32_ragged"),
        # the largest prefill
        _join("join", 16384, 1024, "bf16", "channel", name="join_prefill"),
        # a micro-batch of the f32 layer, gated by token
        _join("join_backward", 1024, 512, "f32", "row", name="join_backward_f32"),
        # a padded micro-batch off every tile: the last norm of a model is not this call's, so nothing follows
        _join("join_backward", 3001, 760, "bf16", "channel", following=False, padding=0.1, name="join_backward_ragged"),
        # a training micro-batch of the largest layer
        _join("join_backward", 16384, 1024, "bf16", "channel", name="join_backward_large"),
        # one small square matrix (an attention output of the default model): all latency
        _matrices("orthogonalize", 1, 512, 512, "f32", name="orthogonalize_one"),
        # unrounded widths of a small model's experts, a bf16 update
        _matrices("orthogonalize", 24, 227, 341, "bf16", name="orthogonalize_ragged"),
        # the default model's experts, gate and up of one layer
        _matrices("muon", 16, 352, 512, "f32", name="muon_default_layer"),
        # down matrices of 16 experts, gradients reduced in bf16
        _matrices("muon", 16, 768, 1408, "bf16", name="muon_down"),
        # gate and up of 64 narrow experts
        _matrices("muon", 128, 704, 1024, "f32", name="muon_fine_grained"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.55:
        while True:
            c = _join(rng.choice(["join", "join", "join_backward"]), _log_int(rng, 1, 16384),
                      rng.choice([512, 768, 1024, _log_int(rng, 64, 2048), 8 * _log_int(rng, 8, 256)]),
                      rng.choice(["bf16", "bf16", "f32"]), rng.choice(["none", "channel", "channel", "row"]),
                      post=rng.random() < 0.75, following=rng.random() < 0.75,
                      padding=rng.choice([0.0, 0.0, 0.1, 0.3]))
            if c["rows"] < 8:
                c["padding"] = 0.0
            if c["rows"] * c["cols"] <= 16384 * 1024 // (2 if c["dtype"] == "f32" else 1):
                return c
    while True:
        rows, cols = (rng.choice([256, 352, 512, 704, 768, 1024, 1408, _log_int(rng, 33, 1408)]) for _ in range(2))
        c = _matrices(rng.choice(["orthogonalize", "muon"]), _log_int(rng, 1, 128), rows, cols, rng.choice(["bf16", "f32"]))
        if work(c)["flops"] <= 7e11 and c["count"] * rows * cols <= 1.0e8:
            return c


# ----------------------------------------------------------------------------- inputs
def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std


class _State:
    pass


def _inputs(case, seed):
    """The tensors that a user's program has in hand before the call."""
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = _State()
    s.case = c
    t = _TORCH[c["dtype"]]
    if c["kind"].startswith("join"):
        r, d = c["rows"], c["cols"]
        s.y = (_normal(g, (r, d)) * (0.2 + 2.0 * torch.rand((r, 1), generator=g, device="cuda"))).to(t)
        s.valid = None
        if c["padding"] > 0:
            s.valid = torch.ones(r, dtype=torch.uint8, device="cuda")
            s.valid[torch.randperm(r, generator=g, device="cuda")[:max(1, round(c["padding"] * r))]] = 0
        s.post = 1.0 + _normal(g, (d,), 0.1) if c["post"] else None
        s.next = 1.0 + _normal(g, (d,), 0.1) if c["following"] else None
        s.gate = None
        if c["gate"] == "channel":
            s.gate = 0.5 + _normal(g, (d,), 0.1)
        elif c["gate"] == "row":
            s.gate = torch.sigmoid(_normal(g, (r, d))).to(t)
        s.scale = 0.22
        s.x = (_normal(g, (r, d)) * 3.0).to(t)  # the residual stream in front of the add, or behind it (backward)
        if c["kind"] == "join_backward":
            s.grad_out = _normal(g, (r, d), 1e-2).to(t)
            s.grad_normed = _normal(g, (r, d), 1e-2).to(t) if c["following"] else None
    else:
        n, r, k = c["count"], c["rows"], c["cols"]
        # a few strong directions (what the rows of a batch have in common) over a broad rest
        strong = torch.matmul(_normal(g, (n, r, 8)), _normal(g, (n, 8, k)))
        s.grad = ((0.3 * strong + _normal(g, (n, r, k))) * 1e-3).to(t)
        if c["kind"] == "muon":
            s.momentum = _normal(g, (n, r, k), 5e-3)
            s.weight = _normal(g, (n, r, k), math.sqrt(2.0 / (r + k)))
            s.lr, s.mu, s.decay = 0.02, 0.95, 0.1
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    c = case
    if own:
        import rustingbrain_amd as rb
        device = _device(rb)
        if c["kind"].startswith("join"):
            s.handle = rb.ResidualJoin(device, c["cols"], dtype=c["dtype"], gate=c["gate"])
            like = lambda v: None if v is None else torch.empty_like(v)  # noqa: E731
            if c["kind"] == "join":
                s.out, s.normed = torch.empty_like(s.x), torch.empty_like(s.x) if c["following"] else None
            else:
                s.grad_x, s.grad_y = torch.empty_like(s.x), torch.empty_like(s.x)
                s.grad_post, s.grad_gate, s.grad_next = like(s.post), like(s.gate), like(s.next)
        else:
            s.handle = rb.Muon(device, c["count"], c["rows"], c["cols"])
            if c["kind"] == "orthogonalize":
                s.out = torch.empty_like(s.grad)
    torch.cuda.synchronize()
    return s


_handle = None


def _device(rb):
    """One handle for the GPU, as a program with many layers keeps."""
    global _handle
    if _handle is None:
        _handle = rb.Device.open(0)
    return _handle


# ----------------------------------------------------------------------------- one pass
def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _rms_inverse(v):
    return torch.rsqrt(v.square().mean(dim=1, keepdim=True) + EPS)


def _join_plain(s):
    x, y = s.x.float(), s.y.float()
    if s.valid is not None:
        y = torch.where(s.valid[:, None] != 0, y, 0.0)
    b = y * _rms_inverse(y) * s.post if s.post is not None else y
    if s.gate is not None:
        b = b * s.gate.float()
    out = (x + s.scale * b).to(s.x.dtype)
    if s.next is None:
        return {"out": out}
    r = out.float()
    return {"out": out, "normed": (r * _rms_inverse(r) * s.next).to(s.x.dtype)}


def _join_backward_plain(s):
    y, total = s.y.float(), s.grad_out.float()
    live = None if s.valid is None else (s.valid[:, None] != 0)
    got = {}
    if s.next is not None:
        r, dn = s.x.float(), s.grad_normed.float()
        k = _rms_inverse(r)
        u = dn * s.next
        total = total + k * u - r * k * k * k * (r * u).mean(dim=1, keepdim=True)
        taken = dn * r * k
        got["grad_next"] = (taken if live is None else torch.where(live, taken, 0.0)).sum(dim=0)
    got["grad_x"] = total.to(s.x.dtype)
    if live is not None:
        y, total = torch.where(live, y, 0.0), torch.where(live, total, 0.0)
    k = _rms_inverse(y) if s.post is not None else None
    n = y * k if s.post is not None else y
    b = n * s.post if s.post is not None else n
    db = s.scale * total
    if s.gate is not None:
        dg = db * b
        got["grad_gate"] = dg.sum(dim=0) if s.case["gate"] == "channel" else dg.to(s.gate.dtype)
        db = db * s.gate.float()
    if s.post is not None:
        got["grad_post"] = (db * n).sum(dim=0)
        v = db * s.post
        db = k * v - y * k * k * k * (y * v).mean(dim=1, keepdim=True)
        if live is not None:
            db = torch.where(live, db, 0.0)
    got["grad_y"] = db.to(s.x.dtype)
    return got


def _orthogonalized(u):
    a, b, c = NS
    x = u / (u.square().sum(dim=(1, 2), keepdim=True).sqrt() + 1e-7)
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.mT.contiguous()
    for _ in range(5):
        g = torch.matmul(x, x.mT.contiguous())
        x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
    return x.mT if tall else x


def _muon_scale(c):
    return math.sqrt(max(1.0, c["rows"] / c["cols"]))


def run(state):
    s, c = state, state.case
    kind = c["kind"]
    if own:
        if kind == "join":
            s.handle.forward_device(c["rows"], _ptr(s.x), _ptr(s.y), _ptr(s.out), _ptr(s.normed), valid_ptr=_ptr(s.valid),
                                    post_weight_ptr=_ptr(s.post), gate_ptr=_ptr(s.gate), next_weight_ptr=_ptr(s.next),
                                    scale=s.scale, eps=EPS)
            return {k: v for k, v in (("out", s.out), ("normed", s.normed)) if v is not None}
        if kind == "join_backward":
            s.handle.backward_device(c["rows"], _ptr(s.y), _ptr(s.x), _ptr(s.grad_out), _ptr(s.grad_normed), _ptr(s.grad_x),
                                     _ptr(s.grad_y), valid_ptr=_ptr(s.valid), post_weight_ptr=_ptr(s.post),
                                     gate_ptr=_ptr(s.gate), next_weight_ptr=_ptr(s.next), scale=s.scale, eps=EPS,
                                     grad_post_ptr=_ptr(s.grad_post), grad_gate_ptr=_ptr(s.grad_gate),
                                     grad_next_ptr=_ptr(s.grad_next))
            got = {"grad_x": s.grad_x, "grad_y": s.grad_y, "grad_post": s.grad_post, "grad_gate": s.grad_gate,
                   "grad_next": s.grad_next}
            return {k: v for k, v in got.items() if v is not None}
        if kind == "orthogonalize":
            s.handle.orthogonalize_device(_ptr(s.grad), _ptr(s.out), dtype=c["dtype"], out_dtype=c["dtype"])
            return s.out
        s.handle.step_device(_ptr(s.grad), _ptr(s.momentum), _ptr(s.weight), dtype=c["dtype"], lr=s.lr, momentum=s.mu,
                             weight_decay=s.decay)
        return {"momentum": s.momentum, "weight": s.weight}
    if kind == "join":
        return _join_plain(s)
    if kind == "join_backward":
        return _join_backward_plain(s)
    if kind == "orthogonalize":
        return _orthogonalized(s.grad.float()).to(s.grad.dtype).contiguous()
    g = s.grad.float()
    s.momentum.mul_(s.mu).add_(g)
    o = _orthogonalized(g + s.mu * s.momentum)
    s.weight.mul_(1.0 - s.lr * s.decay).sub_(s.lr * _muon_scale(c) * o)
    return {"momentum": s.momentum, "weight": s.weight}


# ----------------------------------------------------------------------------- in 64 bits
def _exact_join(s):
    wide = lambda v: None if v is None else v.double()  # noqa: E731
    x, y, gate, post, following = map(wide, (s.x, s.y, s.gate, s.post, s.next))
    norm = lambda v: v / (v.pow(2).sum(1) / v.shape[1] + EPS).sqrt()[:, None]  # noqa: E731
    live = torch.ones(len(x), device=x.device, dtype=torch.float64) if s.valid is None else s.valid.double()
    for v in (y, gate, post, following):
        if v is not None:
            v.requires_grad_()

    def branch():
        b = norm(y * live[:, None]) if post is not None else y * live[:, None]
        b = b if post is None else b * post
        return s.scale * (b if gate is None else b * gate)

    if s.case["kind"] == "join":
        with torch.no_grad():
            out = x + branch()
            got = {"out": out}
            if following is not None:
                got["normed"] = norm(out.to(s.x.dtype).double()) * following
        return got
    # the gradient that reaches the rows behind the add, then what it gives the branch
    with torch.enable_grad():
        stream = x.requires_grad_()
        loss = (stream * s.grad_out.double()).sum()
        got = {}
        if following is not None:
            h = norm(stream)
            (got["grad_next"],) = torch.autograd.grad((h * following * s.grad_normed.double() * live[:, None]).sum(), following,
                                                      retain_graph=True)
            loss = loss + (h * following.detach() * s.grad_normed.double()).sum()
        (total,) = torch.autograd.grad(loss, stream)
        got["grad_x"] = total
        names = [n for n, v in (("grad_y", y), ("grad_post", post), ("grad_gate", gate)) if v is not None]
        leaves = [v for v in (y, post, gate) if v is not None]
        got.update(zip(names, torch.autograd.grad((branch() * total * live[:, None]).sum(), leaves)))
    return got


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"].startswith("join"):
        return _exact_join(s)
    g = s.grad.double()
    if case["kind"] == "muon":
        m = s.momentum.double() * s.mu + g
        g = g + s.mu * m
    a, b, c = NS
    q = g / (torch.linalg.vector_norm(g, dim=(1, 2), keepdim=True) + 1e-7)
    # from the other side, over the longer axis where that is the second: q (a + b G + c G^2) with G = q^T q
    wide = q.shape[2] >= q.shape[1]
    q = q.mT.contiguous() if wide else q
    for _ in range(5):
        h = torch.matmul(q.mT.contiguous(), q)
        q = a * q + b * torch.matmul(q, h) + c * torch.matmul(torch.matmul(q, h), h)
    q = q.mT.contiguous() if wide else q
    if case["kind"] == "orthogonalize":
        return q
    return {"momentum": m, "weight": s.weight.double() * (1.0 - s.lr * s.decay) - s.lr * _muon_scale(case) * q}


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    size = {"f32": 4, "bf16": 2}[c["dtype"]]
    if c["kind"].startswith("join"):
        n = float(c["rows"]) * c["cols"]
        arrays = 3.0 + c["following"] + (c["gate"] == "row")
        parameters = (c["post"] + c["following"] + (c["gate"] == "channel")) * c["cols"] * 4.0
        per = 8.0
        if c["kind"] == "join_backward":
            # y, the gradient behind the add and both input gradients; the rows and their norm's gradient; a row gate's
            arrays = 4.0 + 2.0 * c["following"] + 2.0 * (c["gate"] == "row")
            parameters *= 2.0
            per = 20.0
        return {"bytes": n * arrays * size + parameters + (c["rows"] if c["padding"] > 0 else 0), "flops": per * n}
    n = float(c["count"]) * c["rows"] * c["cols"]
    m, k = min(c["rows"], c["cols"]), max(c["rows"], c["cols"])
    # the product of a matrix with its transpose and the square of a symmetric one: half of either is enough
    flops = 5.0 * c["count"] * (float(m) * m * k + float(m) ** 3 + 2.0 * m * m * k)
    if c["kind"] == "orthogonalize":
        return {"bytes": 2.0 * n * size, "flops": flops}
    return {"bytes": n * (size + 16.0), "flops": flops + 8.0 * n}
