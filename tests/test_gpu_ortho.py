"""Newton-Schulz orthogonalisation and the optimiser step on the GPU against the
definition in 64 bits.

Errors are 2-norms over a whole matrix, relative to the result's.  Allowed, as
derived before the first run: three times the error of the same steps in plain f32
products (the arithmetic the kernels are to match), and at least 3e-5: each of the
five steps makes about 8 roundings of 2^-22 to 2^-24 and hands a perturbation on at
most doubled where the values have saturated, 8 · 2^-23 · (1 + 2 + 4 + 8 + 16).
A 16-bit result adds its rounding: uniform errors of at most half a step, so half a
step over sqrt(3) in this norm (half a step where there are few elements)."""
import math

import pytest
import torch

from spotv2net_amd.graphed import _no_gc

pytestmark = pytest.mark.gpu

NS = (3.4445, -4.7750, 2.0315)
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def definition(g, steps=5, co=NS, eps=1e-7, dtype=torch.float64):
    x = g.to(dtype)
    flip = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if flip else x
    x = x / max(float(g.double().norm()), eps)
    for _ in range(steps):
        s = torch.mm(x, x.t().contiguous())
        x = co[0] * x + torch.mm(co[1] * s + co[2] * torch.mm(s, s), x)
    return x.t().contiguous() if flip else x


def rel(a, r):
    n = float(r.norm())
    d = float((a.double() - r).norm())
    return d / n if n else d


def allowed(g, ref, **kw):
    few = g.numel() < 256
    tol = max(3 * rel(definition(g, dtype=torch.float32, **kw), ref), 3e-5)
    return tol + HALF[g.dtype] / (1.0 if few else math.sqrt(3.0))


def gradient(dev, rows, cols, dtype=torch.float32, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    r = max(1, min(rows, cols) // 4)
    left = torch.randn(rows, r, device=dev, generator=gen) / \
        torch.arange(1, r + 1, device=dev).sqrt()
    g = left @ torch.randn(r, cols, device=dev, generator=gen)
    return (1e-3 * (g + torch.randn(rows, cols, device=dev, generator=gen))).to(dtype)


def check(g, **kw):
    from spotv2net_amd import orthogonalize
    names = {"co": "coefficients"}
    u = orthogonalize(g, **{names.get(k, k): v for k, v in kw.items()})
    assert u.shape == g.shape and u.dtype == g.dtype and u.is_contiguous()
    ref = definition(g, **kw)
    assert rel(u, ref) <= allowed(g, ref, **kw), (tuple(g.shape), rel(u, ref))
    return u


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 130), (30, 30), (31, 33), (64, 64), (65, 64),
          (128, 12), (128, 128), (129, 127), (200, 126), (400, 1260), (1024, 128), (777, 1537),
          (1300, 1300), (1, 4096), (4096, 5), (32, 128), (32, 129), (128, 32), (17, 127), (31, 2049),
          (16384, 3), (32, 5000), (33, 5000)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_against_definition(dev, rows, cols, dtype):
    check(gradient(dev, rows, cols, dtype, seed=rows * 7 + cols))


def test_flat_and_steep_spectra(dev):
    """Singular values all alike (a random matrix), and falling by a thousand."""
    gen = torch.Generator(device=dev).manual_seed(3)
    check(torch.randn(300, 500, device=dev, generator=gen))
    check(torch.randn(500, 300, device=dev, generator=gen).bfloat16())
    q1 = torch.linalg.qr(torch.randn(256, 256, device=dev, generator=gen, dtype=torch.float64))[0]
    q2 = torch.linalg.qr(torch.randn(256, 256, device=dev, generator=gen, dtype=torch.float64))[0]
    s = torch.logspace(0, -3, 256, device=dev, dtype=torch.float64)
    check((torch.mm(q1 * s, q2)).float())


@pytest.mark.parametrize("rows,cols,dtype", [
    (2049, 1999, torch.float32), (16384, 96, torch.float32), (2600, 2570, torch.float32),
    (3000, 3010, torch.float32), (4000, 4100, torch.float32), (4100, 4000, torch.bfloat16),
    (2500, 3100, torch.bfloat16), (1100, 16000, torch.bfloat16)])
def test_large(dev, rows, cols, dtype):
    """Sizes past one round of 128 x 128 tiles, whole and with a remainder."""
    check(gradient(dev, rows, cols, dtype))


def test_large_stack(dev):
    from spotv2net_amd import orthogonalize
    g = torch.stack([gradient(dev, 1500, 1700, seed=k) for k in range(4)])
    u = orthogonalize(g)
    for k in range(4):
        ref = definition(g[k])
        assert rel(u[k], ref) <= allowed(g[k], ref), k


def test_bf16_keeps_its_precision(dev):
    """The bf16 path's cheaper first steps: the result is within 1.1 of what rounding
    the exact one costs (2-norm), on flat, falling and nearly low-rank spectra."""
    from spotv2net_amd import orthogonalize
    gen = torch.Generator(device=dev).manual_seed(21)
    for m, n in ((128, 300), (200, 3000), (512, 512), (1024, 1100), (1300, 5000)):
        noise = torch.randn(m, n, device=dev, generator=gen)
        low = torch.randn(m, 8, device=dev, generator=gen) @ \
            torch.randn(8, n, device=dev, generator=gen)
        for g in (noise, low + 0.05 * noise, gradient(dev, m, n)):
            g = g.bfloat16()
            ref = definition(g)
            assert rel(orthogonalize(g), ref) <= 1.1 * rel(ref.bfloat16(), ref), (m, n)


@pytest.mark.parametrize("co,steps", [((1.5, -0.5, 0.0), 20), ((15 / 8, -10 / 8, 3 / 8), 14)])
def test_other_coefficients_converge(dev, co, steps):
    """Polynomials with a fixed point at 1 give the orthogonal factor itself."""
    gen = torch.Generator(device=dev).manual_seed(9)
    g = torch.randn(60, 150, device=dev, generator=gen)
    from spotv2net_amd import orthogonalize
    u = orthogonalize(g, steps=steps, coefficients=co).double()
    eye = torch.eye(60, device=dev, dtype=torch.float64)
    assert float((torch.mm(u, u.t().contiguous()) - eye).abs().max()) <= 1e-5
    p, _, vh = torch.linalg.svd(g.double(), full_matrices=False)
    assert rel(u, torch.mm(p, vh)) <= 1e-5


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6])
def test_step_counts(dev, steps):
    check(gradient(dev, 70, 200), steps=steps)
    check(gradient(dev, 700, 900), steps=steps)


@pytest.mark.parametrize("batch,rows,cols", [(1, 40, 50), (5, 33, 70), (3, 300, 140), (17, 16, 16), (9, 3, 700), (4, 1500, 30),
                                             (2, 800, 1100)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_stacks_are_their_matrices(dev, batch, rows, cols, dtype):
    from spotv2net_amd import orthogonalize
    g = torch.stack([gradient(dev, rows, cols, dtype, seed=k) * 10.0 ** (k % 5 - 2)
                     for k in range(batch)])
    u = orthogonalize(g)
    assert u.shape == g.shape
    for k in range(batch):
        ref = definition(g[k])
        assert rel(u[k], ref) <= allowed(g[k], ref), k


def test_strides(dev):
    from spotv2net_amd import orthogonalize
    big = gradient(dev, 130, 220)
    base = orthogonalize(big[3:103, 7:190].contiguous())
    assert torch.equal(orthogonalize(big[3:103, 7:190]), base)           # wider rows, odd start
    t = big[3:103, 7:190].contiguous().t()
    assert torch.equal(orthogonalize(t), orthogonalize(t.contiguous()))
    st = gradient(dev, 60, 80).view(4, 15, 80)
    want = orthogonalize(st[::2].contiguous())
    assert torch.equal(orthogonalize(st[::2]), want)                     # every other matrix
    assert torch.equal(orthogonalize(st.transpose(0, 1)[:, ::2]),
                       orthogonalize(st.transpose(0, 1)[:, ::2].contiguous()))
    row = gradient(dev, 1, 80).expand(15, 80)                            # one row repeated
    assert torch.equal(orthogonalize(row), orthogonalize(row.contiguous()))
    mats = gradient(dev, 15, 80).expand(3, 15, 80)                       # one matrix repeated
    u = orthogonalize(mats)
    assert torch.equal(u[0], u[1]) and torch.equal(u[0], u[2])


def test_scale_does_not_matter(dev):
    """Powers of two of the input give the same bits, up to squares that overflow or
    vanish in f32; below eps the result is G / eps carried through the steps."""
    from spotv2net_amd import orthogonalize
    g = gradient(dev, 90, 140)
    u = orthogonalize(g)
    for k in (-10, 30, 90, 120):
        assert torch.equal(orthogonalize(g * 2.0 ** k), u)
    assert torch.equal(orthogonalize(g * 2.0 ** -90, eps=1e-44), u)
    # X_0 = G / eps has a norm far below 1 here: its entries are held to half of 2^-24
    # at a scale of 2^14, which the steps multiply by at most a^5
    small = g * 2.0 ** -40
    ref = definition(small)
    room = 3e-5 * float(ref.norm()) + 2 * NS[0] ** 5 * 2.0 ** -39 * math.sqrt(g.numel())
    assert float((orthogonalize(small).double() - ref).norm()) <= room
    assert not orthogonalize(torch.zeros(40, 70, device=dev)).any()


def test_nonfinite_and_empty(dev):
    from spotv2net_amd import orthogonalize
    g = gradient(dev, 40, 70)
    g[3, 5] = float("nan")
    assert orthogonalize(g).isnan().all()
    g[3, 5] = float("inf")
    assert orthogonalize(g).isnan().any()
    st = torch.stack([gradient(dev, 40, 70), g, gradient(dev, 40, 70, seed=1)])
    u = orthogonalize(st)
    assert torch.equal(u[0], orthogonalize(st[0])) and torch.equal(u[2], orthogonalize(st[2]))
    for shape in ((0, 5), (5, 0), (0, 3, 4), (2, 0, 4)):
        assert orthogonalize(torch.empty(shape, device=dev)).shape == shape


def test_refusals(dev):
    from spotv2net_amd import muon_step, orthogonalize
    g = gradient(dev, 8, 8)
    for bad, msg in ((g.double(), "float32, bfloat16 or float16"), (g[0], "a matrix or a stack"),
                     (torch.empty(16385, 2, device=dev), "sides up to")):
        with pytest.raises(RuntimeError, match=msg):
            orthogonalize(bad)
    for kw, msg in ((dict(steps=0), "steps"), (dict(steps=33), "steps"), (dict(eps=0.0), "eps"),
                    (dict(coefficients=(9.0, 0.0, 0.0)), "grow"),
                    (dict(coefficients=(float("nan"), 0.0, 0.0)), "finite")):
        with pytest.raises(RuntimeError, match=msg):
            orthogonalize(g, **kw)
    w, b = gradient(dev, 8, 8, seed=1), torch.zeros(8, 8, device=dev)
    for args, msg in ((([w, w], [g, g], [b, b.clone()]), "shares memory"),
                      (([w], [w], [b]), "shares memory"), (([w], [g], [w]), "shares memory"),
                      (([w], [g[:4]], [b]), "gradient"), (([w], [g], [b, b]), "different lengths"),
                      (([w.t()], [g], [b]), "contiguous"), (([w], [g.bfloat16()], [b]), "float32"),
                      (([w], [g], [b.cpu()]), "device")):
        with pytest.raises(RuntimeError, match=msg):
            muon_step(*args, lr=0.1)
    for kw in (dict(lr=float("nan")), dict(lr=0.1, weight_decay=float("inf"))):
        with pytest.raises(RuntimeError, match="must be finite"):
            muon_step([w], [g], [b], **kw)
    with pytest.raises(RuntimeError, match="momentum must be"):
        muon_step([w], [g], [b], lr=0.1, momentum=1.0)
    with pytest.raises(ValueError, match="matrices"):
        muon_step([w[0]], [g[0]], [b[0]], lr=0.1)


def muon_reference(ws, gs, ms, lr, momentum=0.95, nesterov=True, weight_decay=0.0, adjust="original"):
    out_w, out_m, upd = [], [], []
    for w, g, m in zip(ws, gs, ms):
        m = momentum * m.double() + (1 - momentum) * g.double()
        u = (1 - momentum) * g.double() + momentum * m if nesterov else m
        rows, cols = w.shape
        f = math.sqrt(max(1.0, rows / cols)) if adjust == "original" else \
            0.2 * math.sqrt(max(rows, cols))
        d = lr * f * definition(u)
        out_w.append((1 - lr * weight_decay) * w.double() - d)
        out_m.append(m)
        upd.append(d)
    return out_w, out_m, upd


def muon_check(ws, gs, ms, refs, steps=1):
    """The momentum within 4 roundings of f32; the weight within 4 of its own and 1e-4
    of the update for every step taken (a bound on f32 Newton-Schulz errors at these
    sizes: the flat spectra above stay under 1e-5 plain)."""
    for w, m, rw, rm, d in zip(ws, ms, *refs):
        assert float((m.double() - rm).norm()) <= 4 * steps * 2.0 ** -24 * float(rm.norm())
        assert float((w.double() - rw).norm()) <= \
            steps * (4 * 2.0 ** -24 * float(rw.norm()) + 1e-4 * float(d.norm()))


def matrices(dev, shapes, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    ws = [torch.randn(m, n, device=dev, generator=gen) / math.sqrt(n) for m, n in shapes]
    gs = [gradient(dev, m, n, seed=seed + 10 + k) for k, (m, n) in enumerate(shapes)]
    ms = [gradient(dev, m, n, seed=seed + 90 + k) for k, (m, n) in enumerate(shapes)]
    return ws, gs, ms


MODELS = [[(8, 8)], [(1, 1)], [(1, 5), (5, 1)], [(400, 1260), (400, 126), (200, 400), (200, 126)],
          [(128, 1024), (128, 12), (128, 128), (128, 12), (128, 128), (128, 12)],
          [(33, 65)] * 16, [(700, 900), (5, 3000), (900, 31), (32, 32)],
          [(1500, 1600), (3, 1600), (1600, 40), (2000, 1)], [(20 + k, 60 - k) for k in range(35)], [(900, 1500), (3, 2)]]


@pytest.mark.parametrize("shapes", MODELS, ids=lambda s: f"{len(s)}x{s[0][0]}x{s[0][1]}")
@pytest.mark.parametrize("kw", [dict(), dict(nesterov=False, weight_decay=0.1),
                                dict(momentum=0.0, adjust="match_rms_adamw", weight_decay=0.5)])
def test_muon_step(dev, shapes, kw):
    from spotv2net_amd import muon_step
    ws, gs, ms = matrices(dev, shapes)
    refs = muon_reference(ws, gs, ms, 0.02, **kw)
    keep = [g.clone() for g in gs]
    kw = dict(kw)
    if "adjust" in kw:
        kw["adjust_lr"] = kw.pop("adjust")
    muon_step(ws, gs, ms, lr=0.02, **kw)
    muon_check(ws, gs, ms, refs)
    assert all(torch.equal(a, b) for a, b in zip(gs, keep))


def test_muon_views_and_neighbours(dev):
    """Weights, momenta and gradients as views of flat buffers at odd offsets: nothing
    beside them is written."""
    from spotv2net_amd import muon_step
    shapes = [(13, 31), (50, 7), (64, 64)]
    n = sum(m * k for m, k in shapes)
    flat = [torch.randn(n + 8, device=dev) for _ in range(3)]
    before = [f.clone() for f in flat]
    views = [[], [], []]
    off = 3
    for m, k in shapes:
        for f, v in zip(flat, views):
            v.append(f[off:off + m * k].view(m, k))
        off += m * k
    refs = muon_reference(*views, 0.05, weight_decay=0.1)
    muon_step(*views, lr=0.05, weight_decay=0.1)
    muon_check(*views, refs)
    for f, b in zip(flat, before):
        assert torch.equal(f[:3], b[:3]) and torch.equal(f[off:], b[off:])
    assert torch.equal(flat[1], before[1])


def test_optimizer_trains_and_resumes(dev):
    """Muon over several steps against the definition; a parameter without a gradient
    is left alone; state_dict carries the momentum."""
    from spotv2net_amd import Muon
    ws, _, _ = matrices(dev, [(40, 90), (90, 40), (16, 16)])
    ps = [torch.nn.Parameter(w.clone()) for w in ws]
    opt = Muon(ps, lr=0.02, weight_decay=0.1)
    ref_w, ref_m = [w.double() for w in ws[:2]], [torch.zeros_like(w).double() for w in ws[:2]]
    total = [0.0, 0.0]
    for k in range(3):
        gs = [gradient(dev, *p.shape, seed=40 + 3 * k + i) for i, p in enumerate(ps)]
        for p, g in zip(ps[:2], gs):
            p.grad = g.t().contiguous().t() if k == 1 else g   # a gradient of another layout
        ref_w, ref_m, upd = muon_reference(ref_w, gs[:2], ref_m, 0.02, weight_decay=0.1)
        total = [t + float(u.norm()) for t, u in zip(total, upd)]
        opt.step()
        if k == 1:
            sd = opt.state_dict()
            opt = Muon(ps, lr=0.5)
            opt.load_state_dict(sd)
    for p, w, t in zip(ps, ref_w, total):
        assert float((p.detach().double() - w).norm()) <= 12 * 2.0 ** -24 * float(w.norm()) + 1e-4 * t
    assert torch.equal(ps[2], ws[2]) and ps[2] not in opt.state


def test_same_bits_every_run(dev):
    from spotv2net_amd import orthogonalize
    for shape in ((300, 500), (60, 2000), (1500, 1400)):
        g = gradient(dev, *shape)
        assert torch.equal(orthogonalize(g), orthogonalize(g))


def test_replayed_graphs(dev):
    """Two captured steps over the same weights and an orthogonalisation, replayed in
    turn with new gradients between eager calls and synchronisations."""
    from spotv2net_amd import muon_step, orthogonalize
    shapes = [(64, 200), (130, 70), (8, 8)]
    ws, gs, ms = matrices(dev, shapes)
    ew, em = [w.clone() for w in ws], [m.clone() for m in ms]

    def step(a, b):
        muon_step(a, gs, b, lr=0.02, weight_decay=0.1)
        return orthogonalize(gs[0])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step([w.clone() for w in ws], [m.clone() for m in ms])
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with _no_gc(), torch.cuda.graph(g):
            out = step(ws, ms)
        graphs.append((g, out))
    for k in range(6):
        for i, g in enumerate(gs):
            g.copy_(gradient(dev, *shapes[i], seed=200 + 7 * k + i))
        graphs[k % 2][0].replay()
        want = step(ew, em)
        torch.cuda.synchronize()
        assert torch.equal(graphs[k % 2][1], want), k
        for a, b in zip(ws + ms, ew + em):
            assert torch.equal(a, b), k


def test_other_stream(dev):
    from spotv2net_amd import orthogonalize
    g = gradient(dev, 500, 800)
    want = orthogonalize(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [orthogonalize(g) for _ in range(3)]
    here = [orthogonalize(g) for _ in range(3)]     # beside it, with a workspace of its own
    torch.cuda.current_stream().wait_stream(s)
    for u in got + here:
        assert torch.equal(u, want)


def test_opcheck(dev):
    ops = torch.ops.sv2n
    utils = ("test_schema", "test_faketensor")
    g = gradient(dev, 20, 30)
    torch.library.opcheck(ops.orthogonalize, (g, 5, *NS, 1e-7), test_utils=utils)
    ws, gs, ms = matrices(dev, [(20, 30), (8, 8)])
    torch.library.opcheck(ops.muon_step, (ws, gs, ms, [1.0, 1.0], 0.02, 0.95, True, 0.1, 5, *NS,
                                          1e-7), test_utils=utils)


def test_past_32_bit_offsets(dev):
    """Matrices of a stack, and rows of a matrix, more than 2^31 elements apart."""
    from spotv2net_amd import orthogonalize
    far = (1 << 31) + 77
    buf = torch.empty(2 * far + 70 * 90, device=dev, dtype=torch.bfloat16)
    st = torch.as_strided(buf, (3, 70, 90), (far, 90, 1))
    g = gradient(dev, 3 * 70, 90, torch.bfloat16).view(3, 70, 90)
    st.copy_(g)
    assert torch.equal(orthogonalize(st), orthogonalize(g))
    rows = torch.as_strided(buf, (3, 90), (far, 1))
    assert torch.equal(orthogonalize(rows), orthogonalize(rows.contiguous()))
    rows = torch.as_strided(buf, (3, 2), (far, 1))
    assert torch.equal(orthogonalize(rows), orthogonalize(rows.contiguous()))


def test_autograd_notices_the_update(dev):
    """A weight saved for a backward and then stepped: the backward refuses."""
    from spotv2net_amd import muon_step
    w = gradient(dev, 8, 8).requires_grad_()
    y = (w * w).sum()
    muon_step([w], [gradient(dev, 8, 8, seed=1)], [torch.zeros(8, 8, device=dev)], lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference_tensors(dev):
    """Tensors of inference mode have no version: stepped like others."""
    from spotv2net_amd import muon_step
    w, g = gradient(dev, 8, 8), gradient(dev, 8, 8, seed=1)
    want, m = w.clone(), torch.zeros(8, 8, device=dev)
    muon_step([want], [g], [m], lr=0.1)
    with torch.inference_mode():
        got, m = w.clone(), torch.zeros(8, 8, device=dev)
        muon_step([got], [g], [m], lr=0.1)
    assert torch.equal(got, want)


def test_first_step_is_not_captured(dev, monkeypatch):
    from spotv2net_amd import Muon
    p = torch.nn.Parameter(gradient(dev, 8, 8))
    p.grad = gradient(dev, 8, 8, seed=1)
    opt = Muon([p], lr=0.1)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="one step before"):
            opt.step()
    opt.step()
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        opt.step()


def test_captured_large_products(dev):
    """The kernels of large and of thin matrices in one captured step, replayed."""
    from spotv2net_amd import muon_step
    shapes = [(1500, 1600), (9, 3000), (40, 300), (6, 6)]
    ws, gs, ms = matrices(dev, shapes)
    ew, em = [w.clone() for w in ws], [m.clone() for m in ms]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        muon_step([w.clone() for w in ws], gs, [m.clone() for m in ms], lr=0.02)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with _no_gc(), torch.cuda.graph(graph):
        muon_step(ws, gs, ms, lr=0.02)
    for k in range(3):
        for i, g in enumerate(gs):
            g.copy_(gradient(dev, *shapes[i], seed=300 + 7 * k + i))
        graph.replay()
        muon_step(ew, gs, em, lr=0.02)
        torch.cuda.synchronize()
        for a, b in zip(ws + ms, ew + em):
            assert torch.equal(a, b), k
