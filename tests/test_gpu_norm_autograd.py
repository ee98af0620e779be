"""layer_norm under what torch's autograd offers besides a plain backward: checkpointing,
saved-tensor hooks, hooks on results and in-place changes of them.  Two runs of the same
kernels over the same numbers give the same bits."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


def leaves(dev, rows=37, cols=60, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    shapes = ((rows, cols), (cols,), (cols,))
    return [torch.randn(*s, device=dev, generator=gen).requires_grad_() for s in shapes]


def plain(fn, xs):
    y = fn(*xs)
    return [y.detach()] + list(torch.autograd.grad((y * y).sum(), xs))


def same(a, b):
    assert len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("where", ["last", "first", "only", "middle"])
@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpoint(dev, where, reentrant):
    """The recomputation runs where the saved rows are first asked for, which is in the
    norm's own backward where it comes last."""
    from spotv2net_amd import layer_norm
    fns = {"last": lambda x, w, b: layer_norm(torch.tanh(x) * w, w, b),
           "first": lambda x, w, b: torch.tanh(layer_norm(x, w, b)) * w,
           "only": layer_norm,
           "middle": lambda x, w, b: layer_norm(torch.tanh(layer_norm(x * 2, w, b)), w, b) * b}
    xs = leaves(dev)
    want = plain(fns[where], xs)
    y = checkpoint(fns[where], *xs, use_reentrant=reentrant)
    for t in xs:
        t.grad = None
    (y * y).sum().backward()
    same([y.detach()] + [t.grad for t in xs], want)


def test_checkpointed_module(dev):
    from spotv2net_amd import LayerNorm
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(24, 40), torch.nn.Tanh(), LayerNorm(40)).to(dev)
    x = torch.randn(50, 24, device=dev)
    grads = []
    for run in (net, lambda t: checkpoint(net, t, use_reentrant=False)):
        net.zero_grad()
        run(x).square().sum().backward()
        grads.append([p.grad.clone() for p in net.parameters()])
    same(*grads)


def test_saved_tensor_hooks(dev):
    from spotv2net_amd import layer_norm
    xs = leaves(dev)
    want = plain(layer_norm, xs)
    with torch.autograd.graph.save_on_cpu():
        y = layer_norm(*xs)
    same([y.detach()] + list(torch.autograd.grad((y * y).sum(), xs)), want)


def test_result_changed_in_place(dev):
    from spotv2net_amd import layer_norm
    xs = leaves(dev)
    want = plain(lambda *a: layer_norm(*a) * 3.0, xs)
    y = layer_norm(*xs)
    y.mul_(3.0)
    same([y.detach()] + list(torch.autograd.grad((y * y).sum(), xs)), want)
