"""Parameters that two layers share: their gradient is the sum of both uses, once.

The two uses' gradients are added in the kernels' buffer here and by the test there, both
in f32: off by a few roundings of the larger one."""
import copy

import pytest
import torch

from helpers import assert_close
from test_gpu_norm_muon_train import build

pytestmark = pytest.mark.gpu


def tie(model, what):
    if what == "norms":
        model.norms[2] = model.norms[1]
    elif what == "norm weights":
        model.norms[1].weight = model.norms[0].weight
    elif what == "layers":
        model.gat_layers[2] = model.gat_layers[1]
    else:
        model.gat_layers[2].lin_src.weight = model.gat_layers[1].lin_src.weight
        model.gat_layers[2].att_src = model.gat_layers[1].att_src
    return model


def test_replayed_graphs(dev):
    """Layers used twice in the plain loop: its replayed graphs against eager runs."""
    from spotv2net_amd import GATModel, synthetic_batch
    torch.manual_seed(0)
    model = GATModel(60, 6, 4, 1, [8, 8, 8, 8], concat_heads=True).to(dev).train()
    model.gat_layers[2] = model.gat_layers[1]
    data = synthetic_batch(3, 2, seed=5, device=dev)
    model.graph_replay = False
    want = torch.autograd.grad(model(data).sum(), list(model.parameters()))
    model.graph_replay = True
    for _ in range(5):
        got = torch.autograd.grad(model(data).sum(), list(model.parameters()))
        for (k, _), a, b in zip(model.named_parameters(), got, want):
            assert_close(a, b, tol=1e-5, what=k)


@pytest.mark.parametrize("what", ["norms", "norm weights", "layers", "layer weights"])
@pytest.mark.parametrize("direct", [False, True])
@pytest.mark.parametrize("n", [30, 40])
def test_shared_parameters(dev, what, direct, n):
    from spotv2net_amd import synthetic_batch
    from spotv2net_amd.stack import direct_grad_accumulation
    model, _ = build(dev, hidden=(8, 8, 8, 8), act="tanh", seed=3, n=n)
    model = tie(model, what)
    names = dict(model.named_parameters(remove_duplicate=False))
    apart = copy.deepcopy(model)
    # every name a parameter of its own
    apart.gat_layers = torch.nn.ModuleList([copy.deepcopy(m) for m in apart.gat_layers])
    apart.norms = torch.nn.ModuleList([copy.deepcopy(m) for m in apart.norms])
    data = synthetic_batch(3, 2, n=n, seed=5, device=dev)
    apart(data).sum().backward()
    want = {}
    for k, q in apart.named_parameters():
        p = names[k]
        want[id(p)] = want.get(id(p), 0) + q.grad.double()
    assert len(want) < len(list(apart.parameters()))
    if direct:
        for p in model.parameters():
            p.grad = torch.zeros_like(p)
        with direct_grad_accumulation():
            out = model(data)
        out.sum().backward()
    else:
        model(data).sum().backward()
    for k, p in model.named_parameters():
        assert_close(p.grad, want[id(p)].float(), tol=1e-5, what=k)
