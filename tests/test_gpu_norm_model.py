"""Norm weights of a model that change between a forward and its backward."""
import pytest
import torch

from test_gpu_norm_muon_train import build

pytestmark = pytest.mark.gpu


def test_changed_weight_is_noticed(dev):
    """A norm's weight changed in place after the forward: the backward needs the old one
    and refuses; a bias it does not need, and a weight that is replaced, change nothing."""
    from spotv2net_amd import synthetic_batch
    model, _ = build(dev, hidden=(16, 8), act="tanh", seed=1)
    model.train()
    data = synthetic_batch(3, 2, seed=5, device=dev)
    params = list(model.parameters())
    want = torch.autograd.grad(model(data).sum(), params)
    for l in (0, 1):
        out = model(data).sum()
        with torch.no_grad():
            model.norms[l].weight.mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward()
        with torch.no_grad():
            model.norms[l].weight.mul_(0.5)
    out = model(data).sum()
    bias = model.norms[0].bias.detach().clone()
    with torch.no_grad():
        model.norms[0].bias.add_(1.0)
    got = torch.autograd.grad(out, params)
    with torch.no_grad():
        model.norms[0].bias.copy_(bias)
    out = model(data).sum()
    old = [m.weight for m in model.norms]
    for m in model.norms:
        m.weight.data = m.weight.data * 3.0
    again = torch.autograd.grad(out, params)
    assert all(a is m.weight for a, m in zip(old, model.norms))
    for g in (got, again):
        for a, b in zip(g, want):
            assert torch.equal(a, b)
