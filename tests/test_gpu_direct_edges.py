"""In the direct mode (TrainStep) no node of the model has an edge to a parameter's own
accumulation node: an eager graph that is alive keeps those on its stream, and a captured
backward that reached one would wait for that stream, which ends the process."""
import copy

import pytest
import torch

from test_gpu_norm_muon_train import build

pytestmark = pytest.mark.gpu


def reached(fn):
    """The leaves whose accumulation nodes a graph reaches."""
    seen, todo, out = set(), [fn], []
    while todo:
        f = todo.pop()
        if f is None or f in seen:
            continue
        seen.add(f)
        if hasattr(f, "variable"):
            out.append(f.variable)
        todo += [g for g, _ in f.next_functions]
    return out


@pytest.mark.parametrize("wide", [False, True])
def test_no_edges_to_the_parameters(dev, wide):
    """Forward, and forward with the loss; plain, and outside the direct mode all of them."""
    from spotv2net_amd import synthetic_batch
    from spotv2net_amd.stack import direct_grad_accumulation
    model, _ = build(dev, hidden=(16, 8), act="tanh", seed=1, n=40 if wide else 30)
    model.train()
    model.graph_replay = False
    data = synthetic_batch(3, 2, n=40 if wide else 30, seed=5, device=dev)
    ids = {id(p) for p in model.parameters()}
    for p in model.parameters():
        p.grad = torch.zeros_like(p)
    for run in (lambda: model(data).sum(), lambda: model.mse_loss(data)):
        loss = run()
        assert {id(v) for v in reached(loss.grad_fn)} == ids
        with direct_grad_accumulation():
            loss = run()
        assert not {id(v) for v in reached(loss.grad_fn)} & ids
        want = torch.autograd.grad(run(), list(model.parameters()))
        for p in model.parameters():
            p.grad.zero_()
        loss.backward()
        for p, g in zip(model.parameters(), want):
            assert torch.equal(p.grad, g)


@pytest.mark.parametrize("optimizer", ["sv2n", "muon"])
def test_capture_beside_an_eager_graph(dev, optimizer):
    """A step with a loss of the user's own, captured while an eager graph of the whole
    model is alive, replayed beside eager steps of a twin."""
    from spotv2net_amd import synthetic_batch
    from spotv2net_amd.train import TrainStep
    model, _ = build(dev, hidden=(24, 10), act="tanh", seed=6)
    twin = copy.deepcopy(model)
    data = synthetic_batch(8, 2, seed=3, device=dev)
    model.train(), twin.train()
    keep = model(data)
    kw = dict(lr=5e-3, optimizer=optimizer, loss_fn=lambda a, b: (a - b).abs().mean())
    a = TrainStep(model, data, use_graph=True, **kw)
    b = TrainStep(twin, data, use_graph=False, **kw)
    for k in range(4):
        a()
        b()
        with torch.no_grad():
            model(data)
        torch.cuda.synchronize()
        for (name, p), (_, q) in zip(model.named_parameters(), twin.named_parameters()):
            assert torch.allclose(p, q, rtol=0, atol=1e-6), (k, name)
    assert keep.grad_fn is not None
