"""Layer norm on the GPU against the definition in 64 bits.

Tolerances are bounds on the rounding of the f32 arithmetic (u = 2^-24), derived
before the first run: a row's sum goes through at most 16 additions in a thread,
10 in the tree over its lanes and waves and 2 more, so a mean is off by at most
28u of the mean magnitude, x - mean by 30u of the row's largest |x|, 1/sqrt by
16u plus what the deviations' rounding gives.  An output of fewer bits adds half a
step of its type."""
import pytest
import torch

from spotv2net_amd.graphed import _no_gc

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}  # half a subnormal step


def reference(x, w, b, dy, eps):
    """y, dx, dw, db in 64 bits, and a bound on the error of each."""
    T = x.dtype
    W = w.dtype if w is not None else T if b is None else b.dtype
    xd, g0 = x.double(), dy.double()
    n, C = xd.shape
    wd = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    bd = torch.zeros_like(wd) if b is None else b.double()
    m = xd.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((xd - m) ** 2).mean(1, keepdim=True) + eps)
    z = (xd - m) * r
    y = z * wd + bd
    big = xd.abs().amax(1, keepdim=True) * r
    ez = 64 * U * (big * (1 + z.abs() / 8) + z.abs())
    ey = ez * wd.abs() + 4 * U * (y.abs() + bd.abs()) + HALF[T] * y.abs() + TINY[T]
    g = g0 * wd
    c1, c2 = g.mean(1, keepdim=True), (g * z).mean(1, keepdim=True)
    dx = r * (g - c1 - z * c2)
    ga = g.abs().mean(1, keepdim=True)
    ec2 = 32 * U * (g * z).abs().mean(1, keepdim=True) + (g.abs() * ez).mean(1, keepdim=True)
    er = 32 * U * (1 + big)  # of r, relative
    edx = r * (2 * U * g.abs() + 30 * U * ga + z.abs() * ec2 + (ez + 4 * U * z.abs()) * c2.abs()) \
        + er * r * (g.abs() + c1.abs() + (z * c2).abs()) + HALF[T] * dx.abs() + TINY[T]
    dw, db = (g0 * z).sum(0), g0.sum(0)
    # additions one after the other: a thread's rows, the groups of a block, the partials
    k = n / 256 + 16 + 8 + 64 + 8
    edw = k * U * (g0 * z).abs().sum(0) + (g0.abs() * ez).sum(0) + HALF[W] * dw.abs() + TINY[W]
    edb = k * U * g0.abs().sum(0) + HALF[W] * db.abs() + TINY[W]
    return (y, dx, dw, db), (ey, edx, edw, edb)


def check(name, got, ref, tol):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (name, int(bad.sum()), float((err / tol.clamp_min(1e-300)).max()))


def make(dev, rows, cols, dtype, wdtype, seed=0, pad=0, affine="wb", offset=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    full = torch.randn(rows, cols + pad, device=dev, generator=g)
    full = (full * 1.5 + offset * torch.randn(rows, 1, device=dev, generator=g)).to(dtype)
    x = full[:, :cols]
    w = (1 + 0.3 * torch.randn(cols, device=dev, generator=g)).to(wdtype) if "w" in affine else None
    b = (0.3 * torch.randn(cols, device=dev, generator=g)).to(wdtype) if "b" in affine else None
    dy = torch.randn(rows, cols, device=dev, generator=g).to(dtype)
    return x, w, b, dy


def run(x, w, b, dy, eps=1e-5):
    from spotv2net_amd import layer_norm
    x = x.detach().requires_grad_()
    ps = [p.detach().requires_grad_() if p is not None else None for p in (w, b)]
    y = layer_norm(x, ps[0], ps[1], eps)
    grads = torch.autograd.grad(y, [x] + [p for p in ps if p is not None], dy)
    it = iter(grads[1:])
    return y.detach(), grads[0], next(it) if w is not None else None, \
        next(it) if b is not None else None


def compare(x, w, b, dy, eps=1e-5):
    got = run(x, w, b, dy, eps)
    ref, tol = reference(x, w, b, dy, eps)
    for name, a, r, t in zip(("y", "dx", "dw", "db"), got, ref, tol):
        if a is not None:
            check(name, a, r, t)
    assert got[0].dtype == got[1].dtype == x.dtype and got[0].is_contiguous()
    return got


SHAPES = [(1, 1), (5, 1), (1, 2), (3, 5), (30, 16), (30, 400), (77, 64), (64, 129), (7, 1261),
          (65, 1024), (33, 1029), (260, 513), (17, 4096), (9, 4100), (5, 8192), (6, 8200),
          (2, 16381), (3, 16384), (5000, 128), (70001, 24), (2049, 256)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32),
                                          (torch.bfloat16, torch.float32),
                                          (torch.bfloat16, torch.bfloat16),
                                          (torch.float16, torch.float32),
                                          (torch.float16, torch.float16)])
def test_against_definition(dev, rows, cols, dtype, wdtype):
    compare(*make(dev, rows, cols, dtype, wdtype, seed=rows + cols))


@pytest.mark.parametrize("affine", ["", "w", "b", "wb"])
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32),
                                          (torch.bfloat16, torch.float32)])
def test_optional_weight_and_bias(dev, affine, dtype, wdtype):
    x, w, b, dy = make(dev, 37, 200, dtype, wdtype, affine=affine)
    got = compare(x, w, b, dy)
    for p, g in ((w, got[2]), (b, got[3])):
        assert (p is None) == (g is None) and (g is None or g.dtype == p.dtype)


@pytest.mark.parametrize("pad", [1, 3, 8, 24])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_row_strides(dev, pad, dtype):
    """A column slice of a wider buffer: rows at every alignment, read in place,
    and nothing of the columns beside it in the result."""
    x, w, b, dy = make(dev, 45, 333, dtype, dtype, pad=pad)
    assert x.stride(0) == 333 + pad
    compare(x, w, b, dy)
    full = torch.full((45, 333 + pad), float("nan"), device=dev, dtype=dtype)
    full[:, :333] = x
    y0 = run(x, w, b, dy)
    y1 = run(full[:, :333], w, b, dy)
    for a, c in zip(y0, y1):
        assert torch.equal(a, c)


def test_unaligned_base_and_layouts(dev):
    """A base address at every element, transposed and 3-D inputs, broadcast dy."""
    buf = torch.randn(30 * 401 + 9, device=dev)
    for off in range(5):
        x = buf[off:off + 30 * 401].view(30, 401)
        _, w, b, dy = make(dev, 30, 401, torch.float32, torch.float32)
        compare(x, w, b, dy)
    xt = torch.randn(64, 50, device=dev).t()
    _, w, b, dy = make(dev, 50, 64, torch.float32, torch.float32)
    compare(xt, w, b, dy.t().contiguous().t())
    from spotv2net_amd import layer_norm
    x3 = torch.randn(4, 6, 64, device=dev).transpose(0, 1)
    y = layer_norm(x3, w, b)
    assert y.shape == (6, 4, 64)
    assert torch.equal(y.reshape(24, 64), layer_norm(x3.reshape(24, 64), w, b))
    assert layer_norm(x3[0, 0], w, b).shape == (64,)
    x = torch.randn(50, 64, device=dev).requires_grad_()
    layer_norm(x, w, b).sum().backward()          # dy is an expanded scalar
    ref, tol = reference(x.detach(), w, b, torch.ones(50, 64, device=dev), 1e-5)
    check("dx", x.grad, ref[1], tol[1])
    row = torch.randn(1, 64, device=dev).expand(50, 64)  # a broadcast input
    compare(row, w, b, dy)


def test_hard_rows(dev):
    """Constant rows (the variance is 0), an offset far above the spread, tiny and
    huge values."""
    x, w, b, dy = make(dev, 12, 500, torch.float32, torch.float32)
    x = x.clone()
    x[0] = 0.0
    x[1] = 3.25
    x[2] += 1e4
    x[3] *= 1e-18
    x[4] *= 1e15
    x[5, 7:] = 0.0
    got = compare(x, w, b, dy)
    assert torch.equal(got[0][0], b)


@pytest.mark.parametrize("cols", [100, 3000])
def test_nonfinite_rows_stay_alone(dev, cols):
    x, w, b, dy = make(dev, 20, cols, torch.float32, torch.float32)
    clean = run(x, w, b, dy)
    xb = x.clone()
    xb[3, 5] = float("nan")
    xb[11, 0] = float("inf")
    bad = run(xb, w, b, dy)
    keep = [i for i in range(20) if i not in (3, 11)]
    for k in (0, 1):
        assert torch.equal(clean[k][keep], bad[k][keep])
        assert bad[k][3].isnan().all() and bad[k][11].isnan().any()


def test_no_rows(dev):
    from spotv2net_amd import layer_norm
    x = torch.empty(0, 40, device=dev, requires_grad=True)
    w = torch.ones(40, device=dev, requires_grad=True)
    b = torch.ones(40, device=dev, requires_grad=True)
    y = layer_norm(x, w, b)
    assert y.shape == (0, 40)
    y.sum().backward()
    assert x.grad.shape == (0, 40) and not w.grad.any() and not b.grad.any()


def test_same_bits_every_run_and_only_what_is_asked(dev):
    x, w, b, dy = make(dev, 4097, 400, torch.float32, torch.float32)
    a, c = run(x, w, b, dy), run(x, w, b, dy)
    for p, q in zip(a, c):
        assert torch.equal(p, q)
    ops = torch.ops.sv2n
    _, mean, rstd = ops.layer_norm(x, w, b, 1e-5)
    for need in ((True, False, False), (False, True, False), (False, False, True),
                 (False, False, False), (True, True, True)):
        out = ops.layer_norm_bwd(dy, x, w, mean, rstd, *need)
        for n, o, r in zip(need, out, a[1:]):
            assert (torch.equal(o, r) if n else o.numel() == 0)
    gw, gb = torch.randn(400, device=dev), torch.randn(400, device=dev)
    sw, sb = gw + a[2], gb + a[3]
    dx = ops.layer_norm_bwd_acc(dy, x, w, mean, rstd, gw, gb)
    assert torch.equal(dx, a[1]) and torch.equal(gw, sw) and torch.equal(gb, sb)
    ops.layer_norm_bwd_acc(dy, x, w, mean, rstd, None, gb)
    assert torch.equal(gw, sw) and torch.equal(gb, sb + a[3])


def test_gradient_against_differences(dev):
    """Central differences of the kernel's own forward along a direction.  Allowed:
    the same quotient's own gap to the gradient in 64 bits, and the outputs'
    rounding divided by the step."""
    from spotv2net_amd import layer_norm
    x, w, b, dy = make(dev, 9, 60, torch.float32, torch.float32)
    _, dx, dw, db = run(x, w, b, dy)
    h = 2.0 ** -6
    for which, grad in (("x", dx), ("w", dw), ("b", db)):
        base = {"x": x, "w": w, "b": b}
        v = (torch.randn_like(base[which]) * 4).round() / 4   # base ± h·v is exact enough in f32
        lo, hi = dict(base), dict(base)
        lo[which], hi[which] = base[which] - h * v, base[which] + h * v
        step = (hi[which].double() - lo[which].double())      # the step really taken
        num = [(layer_norm(s["x"], s["w"], s["b"]).double() * dy.double()).sum() for s in (hi, lo)]
        ref = [reference(s["x"], s["w"], s["b"], dy, 1e-5) for s in (hi, lo)]
        want = ((ref[0][0][0] - ref[1][0][0]) * dy.double()).sum()
        exact = reference(x, w, b, dy, 1e-5)
        k = {"x": 1, "w": 2, "b": 3}[which]
        gap = (want - (exact[0][k] * step).sum()).abs()
        room = sum((r[1][0] * dy.double().abs()).sum() for r in ref) + \
            (exact[1][k] * step.abs()).sum() + gap
        assert ((num[0] - num[1]) - (grad.double() * step).sum()).abs() <= room


def test_replayed_graph(dev):
    """Forward and backward in a captured graph, replayed with new inputs between
    eager calls and synchronisations; the eager graph of the same leaves is gone
    before the capture."""
    from spotv2net_amd import layer_norm
    x, w, b, dy = make(dev, 300, 400, torch.float32, torch.float32)
    xs, ws, bs = x.clone().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
    dys = dy.clone()

    def step():
        y = layer_norm(xs, ws, bs)
        return (y.detach(),) + torch.autograd.grad(y, (xs, ws, bs), dys)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with _no_gc(), torch.cuda.graph(g):
        out = step()
    for k in range(4):
        x2, _, _, dy2 = make(dev, 300, 400, torch.float32, torch.float32, seed=50 + k)
        with torch.no_grad():
            xs.copy_(x2)
            dys.copy_(dy2)
        g.replay()
        eager = run(x2, w, b, dy2)
        torch.cuda.synchronize()
        for a, r in zip(out, eager):
            assert torch.equal(a, r), k


def test_capture_beside_an_eager_graph(dev):
    """A backward captured while an eager graph of the same leaf is alive raises; once
    that graph is gone the same capture runs."""
    from spotv2net_amd import layer_norm
    x, w, b, dy = make(dev, 64, 40, torch.float32, torch.float32)
    xs = x.clone().requires_grad_()
    keep = layer_norm(xs, w, b)

    def step():
        return torch.autograd.grad(layer_norm(xs, w, b), xs, dy)[0]

    with pytest.raises(RuntimeError, match="eager graph"):
        with _no_gc(), torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    want = torch.autograd.grad(keep, xs, dy)[0]
    del keep
    g = torch.cuda.CUDAGraph()
    with _no_gc(), torch.cuda.graph(g):
        out = step()
    g.replay()
    assert torch.equal(out, want)


def test_gradient_buffers_must_not_overlap(dev):
    x, w, b, dy = make(dev, 5, 40, torch.float32, torch.float32)
    _, mean, rstd = torch.ops.sv2n.layer_norm(x, w, b, 1e-5)
    buf = torch.zeros(60, device=dev)
    for dw, db in ((buf[:40], buf[:40]), (buf[:40], buf[20:])):
        with pytest.raises(RuntimeError, match="overlap"):
            torch.ops.sv2n.layer_norm_bwd_acc(dy, x, w, mean, rstd, dw, db)


def test_other_stream(dev):
    x, w, b, dy = make(dev, 2000, 777, torch.float32, torch.float32)
    want = run(x, w, b, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(s)
    for a, r in zip(got, want):
        assert torch.equal(a, r)


def test_module_and_refusals(dev):
    from spotv2net_amd import LayerNorm, layer_norm
    torch.manual_seed(0)
    m = LayerNorm(48).to(dev)
    x = torch.randn(10, 48, device=dev, requires_grad=True)
    (m(x) ** 2).sum().backward()
    assert m.weight.grad.shape == (48,) and x.grad.shape == x.shape
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        layer_norm(x.double())
    with pytest.raises(RuntimeError, match="rows of 1 to 16384"):
        layer_norm(torch.empty(2, 16385, device=dev))
    with pytest.raises(RuntimeError, match="for rows of 48"):
        layer_norm(x, torch.ones(47, device=dev))
    with pytest.raises(RuntimeError, match="expected float32 or the input"):
        layer_norm(x, torch.ones(48, device=dev, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="different types"):
        layer_norm(x.bfloat16(), torch.ones(48, device=dev),
                   torch.ones(48, device=dev, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="input on"):
        layer_norm(x, torch.ones(48))
    with pytest.raises(RuntimeError, match="must not be negative"):
        layer_norm(x, eps=-1.0)
    y = layer_norm(x, m.weight, m.bias)
    (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()   # differentiable once


def test_opcheck(dev):
    x, w, b, dy = make(dev, 30, 100, torch.bfloat16, torch.float32)
    ops = torch.ops.sv2n
    utils = ("test_schema", "test_faketensor")
    torch.library.opcheck(ops.layer_norm, (x, w, b, 1e-5), test_utils=utils)
    _, mean, rstd = ops.layer_norm(x, w, b, 1e-5)
    for need in ((True, True, True), (False, True, False)):
        torch.library.opcheck(ops.layer_norm_bwd, (dy, x, w, mean, rstd, *need), test_utils=utils)
    gw = torch.zeros(100, device=dev)
    torch.library.opcheck(ops.layer_norm_bwd_acc, (dy, x, w, mean, rstd, gw, None),
                          test_utils=utils)


def test_compiles(dev):
    """torch.compile traces the operator and its autograd formula."""
    from spotv2net_amd import layer_norm
    x, w, b, dy = make(dev, 50, 120, torch.float32, torch.float32)
    want = run(x, w, b, dy)

    def f(x, w, b):
        return layer_norm(x * 1.0, w, b) * 1.0

    xs = [t.detach().requires_grad_() for t in (x, w, b)]
    y = torch.compile(f, backend="aot_eager")(*xs)
    got = (y.detach(),) + torch.autograd.grad(y, xs, dy)
    for a, r in zip(got, want):
        assert torch.equal(a, r)


def test_backward_twice(dev):
    """The saved rows go with the first backward unless the graph is kept."""
    from spotv2net_amd import layer_norm
    x, w, b, dy = make(dev, 9, 40, torch.float32, torch.float32)
    xs = x.detach().requires_grad_()
    y = layer_norm(xs, w, b)
    a = torch.autograd.grad(y, xs, dy, retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(y, xs, dy)[0])
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, xs, dy)
    # an input overwritten after the forward is noticed
    xs = x.detach().clone().requires_grad_()
    z = xs * 1.0
    y = layer_norm(z, w, b)
    z.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, xs, dy)


def test_past_32_bit_offsets(dev):
    """More than 2^31 elements: the last rows as if they stood alone."""
    from spotv2net_amd import layer_norm
    rows, cols = 262151, 8200
    x = torch.empty(rows, cols, device=dev, dtype=torch.bfloat16).normal_()
    w = torch.randn(cols, device=dev)
    b = torch.randn(cols, device=dev)
    xs = x.requires_grad_()
    y = layer_norm(xs, w, b)
    (dx,) = torch.autograd.grad(y, xs, x.detach())
    tail = x.detach()[-7:].clone().requires_grad_()
    yt = layer_norm(tail, w, b)
    (dxt,) = torch.autograd.grad(yt, tail, tail.detach())
    assert torch.equal(y[-7:], yt) and torch.equal(dx[-7:], dxt)
