"""layer_norm under torch.func's transforms and asked for gradients of its gradients:
first derivatives as without them, second ones refused and never zero.

Against torch's own layer norm in 64 bits; a first derivative is off by at most 1e-5 of
the largest one (f32 sums of at most 60 terms, of values up to 5)."""
import warnings

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore")]


def own(x, w, b):
    from spotv2net_amd import layer_norm
    return layer_norm(x, w, b)


def ref(x, w, b):
    return torch.nn.functional.layer_norm(x, x.shape[-1:], w, b, 1e-5)


def inputs(dev, rows=9, cols=20):
    gen = torch.Generator(device=dev).manual_seed(4)
    return [torch.randn(*s, device=dev, generator=gen) for s in ((rows, cols), (cols,), (cols,))]


def near(a, b):
    a, b = (t if isinstance(t, tuple) else (t,) for t in (a, b))
    assert len(a) == len(b)
    for p, q in zip(a, b):
        assert p.shape == q.shape
        assert (p.double() - q).abs().max() <= 1e-5 * q.abs().max().clamp_min(1.0)


def loss(f):
    return lambda *a: (f(*a) ** 3).sum()


@pytest.mark.parametrize("argnums", [0, 1, 2, (0, 1, 2)])
def test_grad_and_vjp(dev, argnums):
    xs = inputs(dev)
    x64 = [t.double() for t in xs]
    near(torch.func.grad(loss(own), argnums)(*xs), torch.func.grad(loss(ref), argnums)(*x64))
    dy = torch.randn(9, 20, device=dev)
    near(torch.func.vjp(own, *xs)[1](dy), torch.func.vjp(ref, *x64)[1](dy.double()))


def test_jacobian(dev):
    xs = inputs(dev, 2, 6)
    x64 = [t.double() for t in xs]
    near(torch.func.jacrev(own, (0, 1, 2))(*xs), torch.func.jacrev(ref, (0, 1, 2))(*x64))


def test_vmap(dev):
    x, w, b = inputs(dev)
    xs = torch.stack([x, 2 * x + 1, -x])
    ws = torch.stack([w, b, w * b])
    for dims, args in (((0, None, None), (xs, w, b)), ((None, 0, None), (x, ws, b)),
                       ((0, 0, 0), (xs, ws, ws + 1)), ((1, None, None), (xs.transpose(0, 1), w, b))):
        a64 = [t.double() for t in args]
        near(torch.vmap(own, dims)(*args), torch.vmap(ref, dims)(*a64))
        near(torch.vmap(torch.func.grad(loss(own), (0, 1, 2)), dims)(*args),
             torch.vmap(torch.func.grad(loss(ref), (0, 1, 2)), dims)(*a64))


def test_batched_gradients(dev):
    xs = [t.requires_grad_() for t in inputs(dev, 3, 5)]
    x64 = [t.detach().double().requires_grad_() for t in xs]
    eye = torch.eye(15, device=dev).view(15, 3, 5)
    near(torch.autograd.grad(own(*xs), xs, eye, is_grads_batched=True),
         torch.autograd.grad(ref(*x64), x64, eye.double(), is_grads_batched=True))


@pytest.mark.parametrize("wrt", [0, 1])
def test_second_derivatives_are_refused(dev, wrt):
    xs = inputs(dev)
    first = torch.func.grad(loss(own))
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.func.grad(lambda *a: (first(*a) ** 2).sum(), wrt)(*xs)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.func.jacrev(first)(*xs)
    for fwd in (torch.func.jacfwd(first), torch.func.hessian(loss(own))):
        with pytest.raises(RuntimeError):
            fwd(*xs)
    # of the gradients' argument alone (the gradient is linear in it, its rule absent)
    _, pull = torch.func.vjp(own, *xs)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.func.grad(lambda dy: (pull(dy)[0] ** 2).sum())(torch.ones(9, 20, device=dev))


def test_create_graph(dev):
    """The first derivatives keep their values and refuse a second backward, whichever of
    them and of the inputs it goes through."""
    xs = [t.requires_grad_() for t in inputs(dev)]
    want = torch.autograd.grad(loss(own)(*xs), xs)
    dy = torch.randn(9, 20, device=dev, requires_grad=True)
    for k in range(3):
        grads = torch.autograd.grad(loss(own)(*xs), xs, create_graph=True)
        for g, t in zip(grads, want):
            assert g.requires_grad and torch.equal(g, t)
        with pytest.raises(RuntimeError, match="differentiable once"):
            grads[k].square().sum().backward()
        for t in xs:
            with pytest.raises(RuntimeError, match="differentiable once"):
                grads = torch.autograd.grad(loss(own)(*xs), xs, create_graph=True)
                torch.autograd.grad(grads[k].square().sum(), t)
    x0 = xs[0].detach()
    only_w = torch.autograd.grad(own(x0, xs[1], xs[2]), xs[1:], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        only_w[1].sum().backward()
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        y = own(*xs)
        y.sum().backward(create_graph=True)
    assert xs[0].grad is not None
    for t in xs:
        t.grad = None
