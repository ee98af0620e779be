"""Training steps over a model with frozen parts: what trains moves as the oracle's does,
and nothing of the stack's backward runs where nothing in it trains."""
import pytest
import torch
import torch.nn.functional as F

from helpers import assert_close
from test_gpu_norm_muon_train import build, named

pytestmark = pytest.mark.gpu


def frozen(model, what):
    for k, p in model.named_parameters():
        p.requires_grad_(not k.startswith(what))
    return model


@pytest.mark.parametrize("norms", [False, True])
def test_no_edge_to_a_frozen_stack(dev, norms):
    """The direct mode's node has a gradient only where the eager one has."""
    from spotv2net_amd import GATModel, synthetic_batch
    from spotv2net_amd.stack import direct_grad_accumulation
    model = GATModel(60, 6, 4, 1, [16, 8], concat_heads=True, layer_norm=norms).to(dev).train()
    data = synthetic_batch(2, 2, seed=1, device=dev)
    for what, want in ((("gat_layers", "norms"), False), (("gat_layers.0",), True),
                       (("linear",), True), ((), True)):
        frozen(model, what)
        for p in model.parameters():
            p.grad = torch.zeros_like(p)
        assert model._hidden(data).requires_grad == want
        with direct_grad_accumulation():
            assert model._hidden(data).requires_grad == want, what
    frozen(model, ("gat_layers", "norms"))
    data.x.requires_grad_()
    with direct_grad_accumulation():
        assert model._hidden(data).requires_grad


@pytest.mark.parametrize("optimizer", ["sv2n", "muon"])
@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("own_loss", [False, True])
@pytest.mark.parametrize("what", [("gat_layers", "norms"), ("gat_layers.0", "norms.0"), ("linear",)])
def test_training_with_frozen_parts(dev, optimizer, use_graph, own_loss, what, monkeypatch):
    from spotv2net_amd import stack, synthetic_batch
    from spotv2net_amd.train import TrainStep
    model, ref = build(dev, hidden=(16, 8), act="tanh", seed=4)
    ref = ref.double().train()
    frozen(model.train(), what)
    before = {k: v.clone() for k, v in model.state_dict().items()}
    data = synthetic_batch(6, 2, seed=9)
    loss = F.mse_loss(ref(data.x.double(), data.edge_index, data.edge_attr.double()),
                      data.y_x.double())
    loss.backward()
    calls = []
    run = stack.stack_backward
    monkeypatch.setattr(stack, "stack_backward", lambda *a, **k: (calls.append(1), run(*a, **k))[1])
    kw = dict(loss_fn=lambda a, b: ((a - b) ** 2).mean()) if own_loss else {}
    step = TrainStep(model, data.to(dev), lr=1e-2, use_graph=use_graph, optimizer=optimizer, **kw)
    got = step()
    torch.cuda.synchronize()
    assert abs(float(got) - float(loss.detach())) <= 1e-5 * max(1.0, float(loss.detach()))
    assert bool(calls) == (what[0] != "gat_layers")
    # (Adam's first step is lr times the gradient's sign, Muon's a scaled orthogonal matrix)
    for k, p, q in named(model, ref):
        if not p.requires_grad:
            assert torch.equal(p, before[k]), k
        elif p.dim() != 2 or "linear" in k or optimizer == "sv2n":
            g = q.grad
            sure = g.abs() > 1e-5 * g.abs().max()
            moved = (p - before[k]).cpu().double()
            assert_close(moved[sure], (-1e-2 * g / (g.abs() + 1e-8))[sure], tol=1e-3, what=k)
        else:
            assert not torch.equal(p, before[k]), k
