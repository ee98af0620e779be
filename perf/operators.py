"""Cases that measure the layer norm and the orthogonalised (Newton-Schulz) weight update.

``run`` computes them in plain torch operations; with ``own`` set it makes the calls a training
program makes of ``spotv2net_amd``.  Four kinds of pass:

* ``ln_fwd``:   y = layer_norm(x, w, b), as in inference;
* ``ln_train``: y and the gradients dx, dw, db for a given dy, as in a training step;
* ``ortho``:    U = orthogonalize(G), G a matrix or a stack of matrices;
* ``muon``:     one optimiser step over a model's weight matrices, in place.
"""
import math

import torch

own = False

EPS_LN = 1e-5
EPS_NS = 1e-7
NS = (3.4445, -4.7750, 2.0315)
STEPS = 5
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.1
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _ln(op, rows, cols, dtype, wdtype, pad=0, name=None):
    c = {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "wdtype": wdtype, "pad": pad}
    return dict(c, name=name) if name else c


def _ortho(batch, rows, cols, dtype, name=None):
    c = {"op": "ortho", "batch": batch, "rows": rows, "cols": cols, "dtype": dtype}
    return dict(c, name=name) if name else c


def _muon(shapes, name=None):
    c = {"op": "muon", "shapes": shapes}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one 30-asset graph's hidden features at inference: nothing but latency
        _ln("ln_fwd", 30, 400, "f32", "f32", name="ln_fwd_graph"),
        # 512 graphs of 30 assets, hidden width 4 x 100
        _ln("ln_fwd", 15360, 400, "f32", "f32", name="ln_fwd_512_graphs"),
        # a wide hidden state in bf16, far past the caches
        _ln("ln_fwd", 16384, 8192, "bf16", "f32", name="ln_fwd_wide_bf16"),
        # the training step of 512 graphs of 30 assets
        _ln("ln_train", 15360, 400, "f32", "f32", name="ln_train_512_graphs"),
        # 128 windows of 30 assets, hidden width 6 x 500, bf16 activations and f32 weights
        _ln("ln_train", 3840, 3000, "bf16", "f32", name="ln_train_6x500_bf16"),
        # 1,024 graphs of 256 nodes, hidden width 8 x 16: many short rows
        _ln("ln_train", 262144, 128, "f32", "f32", name="ln_train_256_nodes"),
        # an odd number of odd rows out of a wider buffer, everything in f16
        _ln("ln_train", 10007, 1261, "f16", "f16", pad=3, name="ln_train_odd_f16"),
        # the first projection of the 256-node model: a small wide matrix
        _ortho(1, 128, 1024, "f32", name="ortho_128x1024"),
        # a stack of tall matrices with odd sides
        _ortho(3, 1537, 777, "f32", name="ortho_3_odd"),
        # a large square matrix in bf16
        _ortho(1, 4096, 4096, "bf16", name="ortho_4096_bf16"),
        # every weight matrix of the two-layer model (4 heads of 100 and 50)
        _muon("400x1260,400x126,200x400,200x126", name="muon_two_layers"),
        # the weight matrices of the one-layer model with 6 heads of 500
        _muon("3000x1260,3000x126", name="muon_6x500"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("ln_fwd", "ln_train", "ortho", "muon"))
    if op in ("ln_fwd", "ln_train"):
        cols = _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, min(262144, (16384 * 8192 if op == "ln_fwd" else 262144 * 128) // cols))
        dtype = rng.choice(tuple(DTYPES))
        return _ln(op, rows, cols, dtype, rng.choice(("f32", dtype)), rng.choice((0, 0, 1, 8, 24)))
    if op == "ortho":
        rows, cols = _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)
        batch = rng.choice((1, 1, 2, rng.randint(3, 6)))
        if batch > 1:
            rows, cols = min(rows, 2048), min(cols, 2048)
        return _ortho(batch, rows, cols, rng.choice(tuple(DTYPES)))
    width = _log_int(rng, 8, 2048)
    shapes = ["%dx%d" % (width, _log_int(rng, 8, 2048))]
    for _ in range(rng.randint(0, 5)):
        shapes.append("%dx%d" % (rng.choice((width, _log_int(rng, 8, 2048))), _log_int(rng, 2, 1500)))
    return _muon(",".join(shapes))


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["shapes"].split(",")]


def _gradient(gen, rows, cols):
    """A weight gradient as training gives it: a few directions carry most of it, the rest is
    noise; its size is that of a mean-reduced loss."""
    r = max(1, min(rows, cols) // 4)
    kw = dict(device="cuda", generator=gen)
    left = torch.randn(rows, r, **kw) * torch.arange(1, r + 1, device="cuda").rsqrt()
    return 1e-3 * (left @ torch.randn(r, cols, **kw) + torch.randn(rows, cols, **kw))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(device="cuda", generator=gen)
    op = case["op"]
    if op in ("ln_fwd", "ln_train"):
        rows, cols, pad = case["rows"], case["cols"], case["pad"]
        dt, wt = DTYPES[case["dtype"]], DTYPES[case["wdtype"]]
        # hidden features: of several scales and offsets, a part of them cut off at zero by relu
        full = torch.randn(rows, cols + pad, **kw)
        full = full * torch.empty(1, cols + pad, device="cuda").uniform_(0.5, 2.0, generator=gen)
        full = full + torch.randn(rows, 1, **kw)
        full[:, : (cols + pad) // 2].relu_()
        x = full.to(dt)[:, :cols]
        w = (1 + 0.2 * torch.randn(cols, **kw)).to(wt)
        b = (0.2 * torch.randn(cols, **kw)).to(wt)
        s = {"op": op, "x": x, "w": w, "b": b}
        if op == "ln_train":
            s["dy"] = (torch.randn(rows, cols, **kw) * 0.1).to(dt)
            for k in "xwb":
                s[k].requires_grad_()
        return s
    if op == "ortho":
        g = torch.stack([_gradient(gen, case["rows"], case["cols"]) for _ in range(case["batch"])])
        g = g.to(DTYPES[case["dtype"]])
        return {"op": op, "g": g if case["batch"] > 1 else g[0].clone()}
    shapes = _shapes(case)
    return {"op": op,
            "w": [torch.randn(m, n, **kw) / math.sqrt(n) for m, n in shapes],
            "g": [_gradient(gen, m, n) for m, n in shapes],
            "buf": [_gradient(gen, m, n) for m, n in shapes]}


def _plain_ln(x, w, b):
    x = x.float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = (d.square().mean(1, keepdim=True) + EPS_LN).rsqrt()
    xhat = d * rstd
    return xhat * w.float() + b.float(), xhat, rstd


def _plain_ns(g):
    x = g.float()
    wide = x.shape[-2] <= x.shape[-1]
    x = x if wide else x.mT.contiguous()
    # the norm is a long sum
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = x / norm.clamp_min(EPS_NS).float()
    a, b, c = NS
    for _ in range(STEPS):
        xt = x.mT.contiguous()
        s = x @ xt
        x = a * x + (b * s + c * (s @ s)) @ x
    return x if wide else x.mT


def run(state):
    op = state["op"]
    if own:
        import spotv2net_amd as sv
        if op == "ln_fwd":
            return sv.layer_norm(state["x"], state["w"], state["b"], EPS_LN)
        if op == "ln_train":
            x, w, b = state["x"], state["w"], state["b"]
            y = sv.layer_norm(x, w, b, EPS_LN)
            dx, dw, db = torch.autograd.grad(y, (x, w, b), state["dy"])
            return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
        if op == "ortho":
            return sv.orthogonalize(state["g"], steps=STEPS, coefficients=NS, eps=EPS_NS)
        sv.muon_step(state["w"], state["g"], state["buf"], lr=LR, momentum=MOMENTUM,
                     nesterov=True, weight_decay=DECAY, steps=STEPS, coefficients=NS, eps=EPS_NS)
        return {"w": state["w"], "buf": state["buf"]}
    with torch.no_grad():
        if op == "ln_fwd":
            return _plain_ln(state["x"], state["w"], state["b"])[0].to(state["x"].dtype)
        if op == "ln_train":
            x, w, b, dy = state["x"], state["w"], state["b"], state["dy"].float()
            y, xhat, rstd = _plain_ln(x, w, b)
            wdy = dy * w.float()
            m1 = wdy.mean(1, keepdim=True)
            m2 = (wdy * xhat).mean(1, keepdim=True)
            dx = rstd * (wdy - m1 - xhat * m2)
            return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": (dy * xhat).sum(0).to(w.dtype),
                    "db": dy.sum(0).to(b.dtype)}
        if op == "ortho":
            return _plain_ns(state["g"]).to(state["g"].dtype).contiguous()
        for w, g, buf in zip(state["w"], state["g"], state["buf"]):
            buf.mul_(MOMENTUM).add_(g * (1 - MOMENTUM))
            u = _plain_ns(g * (1 - MOMENTUM) + buf * MOMENTUM)
            w.mul_(1 - LR * DECAY)
            w.sub_(u * (LR * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))))
        return {"w": state["w"], "buf": state["buf"]}


def _ns_flops(m, n):
    """Multiply-adds x 2 of the steps: S = X Xt and S S are symmetric (half is enough), then
    (b S + c S S) X; m <= n."""
    m, n = min(m, n), max(m, n)
    return STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)


def work(case):
    op = case["op"]
    if op in ("ln_fwd", "ln_train"):
        e = DTYPES[case["dtype"]].itemsize * case["rows"] * case["cols"]
        w = DTYPES[case["wdtype"]].itemsize * case["cols"]
        if op == "ln_fwd":
            return {"bytes": 2 * e + 2 * w, "flops": 8 * case["rows"] * case["cols"]}
        # reads x, dy, w, b; writes y, dx, dw, db (x is read once for the pass as a whole)
        return {"bytes": 4 * e + 4 * w, "flops": 20 * case["rows"] * case["cols"]}
    if op == "ortho":
        m, n = case["rows"], case["cols"]
        return {"bytes": 2 * case["batch"] * m * n * DTYPES[case["dtype"]].itemsize,
                "flops": case["batch"] * _ns_flops(m, n)}
    sizes = _shapes(case)
    # reads the weight, the gradient and the momentum, writes the weight and the momentum
    return {"bytes": sum(20 * m * n for m, n in sizes), "flops": sum(_ns_flops(m, n) for m, n in sizes)}


def _exact_ns(g):
    """f(G) = P G with P a polynomial in the smaller Gram matrix K: with A_k = P_k K P_k,
    P_0 = I / |G| and P_{k+1} = (a I + b A_k + c A_k A_k) P_k."""
    g = g.double()
    flip = g.shape[0] > g.shape[1]
    h = g.t() if flip else g
    k = torch.mm(h, h.t().contiguous())
    eye = torch.eye(k.shape[0], dtype=torch.float64, device=g.device)
    p = eye / max(math.sqrt(float(torch.trace(k))), EPS_NS)
    for _ in range(STEPS):
        s = torch.mm(torch.mm(p, k), p)
        p = torch.mm(NS[0] * eye + torch.mm(NS[1] * eye + NS[2] * s, s), p)
    u = torch.mm(p, h.contiguous())
    return u.t().contiguous() if flip else u


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op in ("ln_fwd", "ln_train"):
            x, w, b = (s[k].detach().double() for k in "xwb")
            n = x.shape[1]
            sigma2 = torch.var(x, 1, unbiased=False, keepdim=True) + EPS_LN
            z = (x - torch.sum(x, 1, keepdim=True) / n) / torch.sqrt(sigma2)
            y = torch.addcmul(b, z, w)
            if op == "ln_fwd":
                return y
            dy = s["dy"].double()
            dz = dy * w
            # the projection of dz / sigma off the directions 1 and z
            dx = (n * dz - dz.sum(1, keepdim=True) - z * (z * dz).sum(1, keepdim=True))
            dx = dx / (n * torch.sqrt(sigma2))
            return {"y": y, "dx": dx, "dw": torch.sum(z * dy, 0), "db": torch.sum(dy, 0)}
        if op == "ortho":
            g = s["g"]
            return torch.stack([_exact_ns(v) for v in g]) if g.dim() == 3 else _exact_ns(g)
        ws, bufs = [], []
        for w, g, buf in zip(s["w"], s["g"], s["buf"]):
            g64 = g.double()
            m = MOMENTUM * buf.double() + (1 - MOMENTUM) * g64
            u = _exact_ns((1 - MOMENTUM) * g64 + MOMENTUM * m)
            scale = LR * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
            ws.append((1 - LR * DECAY) * w.double() - scale * u)
            bufs.append(m)
        return {"w": ws, "buf": bufs}
