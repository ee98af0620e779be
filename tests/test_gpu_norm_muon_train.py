"""Layer norm inside GATModel and Muon inside TrainStep: the model against the oracle
with layer norms between its layers, and training steps that use both against a
restatement in 64 bits."""
import copy
import math

import pytest
import torch
import torch.nn.functional as F

from helpers import assert_close, assert_parity, block_graphs, float64_twin

pytestmark = pytest.mark.gpu

NS = (3.4445, -4.7750, 2.0315)


class NormedOracle(torch.nn.Module):
    """The oracle's layers with torch's layer norm on every layer's output."""

    def __init__(self, model, kw):
        super().__init__()
        from oracle.pyg_gatconv import OracleGATModel
        self.net = OracleGATModel(**kw)
        sd = {k: v.cpu() for k, v in model.state_dict().items() if not k.startswith("norms")}
        self.net.load_state_dict(sd)
        self.norms = torch.nn.ModuleList([torch.nn.LayerNorm(m.normalized_shape) for m in model.norms])
        self.norms.load_state_dict({k[6:]: v.cpu() for k, v in model.state_dict().items()
                                    if k.startswith("norms")})

    def forward(self, x, edge_index, edge_attr):
        for conv, norm in zip(self.net.gat_layers, self.norms):
            x = norm(self.net.a(conv(x, edge_index, edge_attr)))
        return self.net.linear(x).view(-1)


def build(dev, S=2, n=30, hidden=(16, 8), heads=4, act="tanh", seed=0, **kw):
    from spotv2net_amd import GATModel
    kw = dict(num_node_features=n * S, num_edge_features=3 * S, num_heads=heads,
              output_node_channels=1, dim_hidden_layers=list(hidden), concat_heads=True,
              activation=act, **kw)
    torch.manual_seed(seed)
    model = GATModel(layer_norm=True, **kw)
    with torch.no_grad():
        for m in model.norms:
            m.weight.add_(0.2 * torch.randn_like(m.weight))
            m.bias.add_(0.2 * torch.randn_like(m.bias))
    ref = NormedOracle(model, kw)
    return model.to(dev), ref


def named(model, ref):
    """(name, parameter, the oracle's) of everything that trains."""
    own = dict(model.named_parameters())
    for k, q in ref.named_parameters():
        k = k[4:] if k.startswith("net.") else k
        if k in own:
            yield k, own[k], q


@pytest.mark.parametrize("hidden,heads,act,n", [
    ((16, 8), 4, "tanh", 30), ((12,), 3, "sigmoid", 30), ((8, 8, 5), 2, "tanh", 17),
    ((16, 16, 16), 8, "tanh", 40), ((8, 8, 5), 2, "sigmoid", 40), ((33, 7), 1, "sigmoid", 30)])
def test_model_matches_oracle(dev, hidden, heads, act, n):
    """Forward and every gradient, on the n <= 32 and the larger-graph attention."""
    from spotv2net_amd import synthetic_batch
    model, ref = build(dev, n=n, hidden=hidden, heads=heads, act=act)
    data = synthetic_batch(3, 2, n=n, seed=5)
    r64 = float64_twin(ref)
    out = model(data.to(dev))
    want = ref(data.x, data.edge_index, data.edge_attr)
    want64 = r64(data.x.double(), data.edge_index, data.edge_attr.double())
    assert_parity(out, want, want64, what="out")
    dout = torch.randn(out.shape, generator=torch.Generator().manual_seed(1))
    out.backward(dout.to(dev))
    want.backward(dout)
    want64.backward(dout.double())
    g64 = {k: q.grad for k, _, q in named(model, r64)}
    count = 0
    for k, p, q in named(model, ref):
        assert_parity(p.grad, q.grad, g64[k], what=k)
        count += 1
    assert count == len(list(model.parameters()))


def test_relu_and_input_gradient(dev):
    """relu: the activation's backward leaves the product that it is fused into without
    norms; the input's gradient passes through the first layer's norm."""
    from spotv2net_amd import synthetic_batch
    model, ref = build(dev, hidden=(16, 8), act="relu", seed=3)
    data = synthetic_batch(2, 2, seed=8)
    xg = data.x.clone().to(dev).requires_grad_()
    d = data.to(dev)
    d.x = xg
    model(d).sum().backward()
    xr = data.x.clone().requires_grad_()
    ref(xr, data.edge_index, data.edge_attr).sum().backward()
    assert_close(xg.grad, xr.grad, tol=2e-5, what="dx")
    for k, p, q in named(model, ref):
        assert_close(p.grad, q.grad, tol=2e-5, what=k)


def test_bf16_and_other_layouts_run(dev):
    """The bf16 mode near the f32 one, and a shuffled edge order equal to its sorted
    graph's result."""
    from spotv2net_amd import Data, synthetic_batch
    model, _ = build(dev, hidden=(16, 8), act="tanh")
    data = synthetic_batch(4, 2, seed=2).to(dev)
    base = model(data)
    half = copy.deepcopy(model).set_precision("bf16")(data)
    assert_close(half, base, tol=5e-2, what="bf16")
    perm = torch.randperm(data.edge_index.size(1), generator=torch.Generator().manual_seed(0))
    ei = block_graphs(4, 30)[:, perm].contiguous().to(dev)
    shuf = Data(x=data.x, edge_index=ei, edge_attr=data.edge_attr[perm.to(dev)].contiguous())
    shuf.nodes_per_graph = 30
    assert_close(model(shuf), base, what="shuffled")


def test_state_dict_and_modes(dev):
    from spotv2net_amd import GATModel, synthetic_batch
    model, _ = build(dev)
    plain = GATModel(60, 6, 4, 1, [16, 8], concat_heads=True, activation="tanh")
    extra = set(model.state_dict()) - set(plain.state_dict())
    assert extra == {f"norms.{l}.{k}" for l in (0, 1) for k in ("weight", "bias")}
    assert plain.norms is None
    data = synthetic_batch(2, 2, seed=1).to(dev)
    drop, _ = build(dev, dropout=0.5)
    drop.train()
    assert not torch.equal(drop(data), drop(data))
    drop.eval()
    assert torch.equal(drop(data), drop(data))
    # a frozen norm still hands the gradient on
    for p in model.norms.parameters():
        p.requires_grad_(False)
    model(data).sum().backward()
    assert all(p.grad is None for p in model.norms.parameters())
    assert model.gat_layers[0].lin_src.weight.grad.abs().max() > 0


def ns64(g):
    x = g.double()
    flip = x.shape[0] > x.shape[1]
    x = x.t() if flip else x
    x = x / x.norm().clamp_min(1e-7)
    for _ in range(5):
        s = x @ x.t()
        x = NS[0] * x + (NS[1] * s + NS[2] * (s @ s)) @ x
    return x.t() if flip else x


class RefOptimizer:
    """Adam for what is not a matrix of the GAT layers, Muon (the update scaled by 0.2
    sqrt(max(rows, cols))) for those, on the oracle's parameters, in 64 bits."""

    def __init__(self, ref, lr):
        ps = {k: p for k, p in ref.named_parameters()}
        self.mats = [p for k, p in ps.items() if p.dim() == 2 and not k.startswith("net.linear")]
        ids = {id(p) for p in self.mats}
        self.adam = torch.optim.Adam([p for p in ps.values() if id(p) not in ids], lr=lr)
        self.m = [torch.zeros_like(p) for p in self.mats]
        self.lr = lr

    def step(self):
        self.adam.step()
        with torch.no_grad():
            for p, m in zip(self.mats, self.m):
                m.mul_(0.95).add_(p.grad, alpha=0.05)
                u = ns64(0.05 * p.grad + 0.95 * m)
                p.sub_(self.lr * 0.2 * math.sqrt(max(p.shape)) * u)


@pytest.mark.parametrize("use_graph", [False, True])
def test_training_steps_match_restatement(dev, use_graph):
    """Three captured (and eager) steps of a model with norms under Muon: the first
    step's loss to f32, then within what its lr-sized first moves allow."""
    from spotv2net_amd import synthetic_batch
    from spotv2net_amd.train import FlatMuon, TrainStep
    model, ref = build(dev, hidden=(16, 8), act="tanh", seed=4)
    ref = ref.double().train()
    model.train()
    data = synthetic_batch(6, 2, seed=9)
    lr = 1e-2
    step = TrainStep(model, data.to(dev), lr=lr, use_graph=use_graph, optimizer="muon")
    assert isinstance(step.opt, FlatMuon)
    assert len(step.opt.w) == sum(p.dim() == 2 for p in model.gat_layers.parameters())
    for k, p, q in named(model, ref):    # construction trains nothing
        assert_close(p, q, what=k)
    opt = RefOptimizer(ref, lr)
    for k in range(3):
        loss = F.mse_loss(ref(data.x.double(), data.edge_index, data.edge_attr.double()),
                          data.y_x.double())
        for p in ref.parameters():
            p.grad = None
        loss.backward()
        opt.step()
        got = step()
        torch.cuda.synchronize()
        assert abs(float(got) - float(loss.detach())) <= (1e-5 if k == 0 else 1e-3) * max(1.0, float(loss.detach())), k
        if k == 0:
            for name, p, q in named(model, ref):
                if p.dim() == 2 and "linear" not in name:   # U to f32 accuracy, times lr
                    assert_close(p, q, tol=2e-5, what=name)


def test_replays_equal_eager_steps(dev):
    """The captured step replayed beside eager steps of a twin, with an eager forward of
    the same parameters kept alive and evaluated between the replays."""
    from spotv2net_amd import synthetic_batch
    from spotv2net_amd.train import TrainStep
    model, _ = build(dev, hidden=(24, 10), act="relu", seed=6, dropout=0.0)
    twin = copy.deepcopy(model)
    data = synthetic_batch(8, 2, seed=3, device=dev)
    model.train(), twin.train()
    keep = model(data)                       # an eager graph of the same leaves
    a = TrainStep(model, data, lr=5e-3, use_graph=True, optimizer="muon")
    b = TrainStep(twin, data, lr=5e-3, use_graph=False, optimizer="muon")
    for k in range(4):
        a()
        b()
        with torch.no_grad():
            model(data)
        torch.cuda.synchronize()
        for (name, p), (_, q) in zip(model.named_parameters(), twin.named_parameters()):
            assert torch.allclose(p, q, rtol=0, atol=1e-6), (k, name)
    assert keep.grad_fn is not None


@pytest.mark.parametrize("optimizer", ["sv2n", "muon"])
def test_no_collection_while_capturing(dev, optimizer):
    """A graph among the garbage, collected while another is captured, ends the process
    (its destructor synchronises the device): the collector is off meanwhile, and on
    again afterwards."""
    import gc
    from spotv2net_amd import synthetic_batch
    from spotv2net_amd.train import ForwardStep, TrainStep
    model, _ = build(dev, hidden=(7, 5), heads=3, seed=2)
    data = synthetic_batch(2, 2, seed=0, device=dev)
    seen = []

    def prepare():
        if torch.cuda.is_current_stream_capturing():
            seen.append(gc.isenabled())

    TrainStep(model, data, optimizer=optimizer, prepare=prepare)
    ForwardStep(model.eval(), data, prepare=prepare)
    assert seen == [False, False] and gc.isenabled()


def test_flat_layout(dev):
    """Every parameter starts on 16 bytes, the matrices last, values kept."""
    from spotv2net_amd import synthetic_batch
    from spotv2net_amd.train import TrainStep
    model, _ = build(dev, hidden=(7, 5), heads=3, seed=2)
    before = {k: v.clone() for k, v in model.state_dict().items()}
    step = TrainStep(model, synthetic_batch(2, 2, seed=0, device=dev), use_graph=False,
                     optimizer="muon")
    for k, v in model.state_dict().items():
        assert torch.equal(v, before[k]), k
    base = step.flat_params.data_ptr()
    ends = []
    for p in step.params:
        assert (p.data_ptr() - base) % 16 == 0 and p.grad.data_ptr() % 16 == 0
        ends.append((p.dim() == 2 and p is not model.linear.weight, p.data_ptr()))
    assert ends == sorted(ends)


def test_fit_with_muon(dev):
    """The whole loop (gather, graphs, test pass) under Muon with norms: the losses it
    reports are finite and the parameters move."""
    from spotv2net_amd import GATModel, WindowDataset, synthetic_series
    from spotv2net_amd.train import Fit
    torch.manual_seed(0)
    vol, volvol = synthetic_series(60, n=30, seed=1)
    ds = WindowDataset(vol.to(dev), volvol.to(dev), 2)
    model = GATModel(60, 6, 2, 1, [8, 4], concat_heads=True, layer_norm=True, dropout=0.1).to(dev)
    w0 = model.gat_layers[0].lin_src.weight.detach().clone()
    f = Fit(model, ds, 16, lr=1e-3, optimizer="muon")
    for _ in range(2):
        rec = f.run_epoch()
        assert math.isfinite(rec["train_loss"]) and math.isfinite(rec["test_loss"])
    assert not torch.equal(model.gat_layers[0].lin_src.weight, w0)


def test_fit_bf16(dev):
    """The bf16 mode's own layer-0 operands (x gathered as its bf16 twin alone) with a
    norm behind them."""
    from spotv2net_amd import GATModel, WindowDataset, synthetic_series
    from spotv2net_amd.train import Fit
    torch.manual_seed(0)
    vol, volvol = synthetic_series(110, n=30, seed=1)
    ds = WindowDataset(vol.to(dev), volvol.to(dev), 4)
    model = GATModel(120, 12, 6, 1, [64], concat_heads=True, layer_norm=True).to(dev)
    model.set_precision("bf16")
    f = Fit(model, ds, 64, lr=1e-3, optimizer="muon")
    a, b = f.run_epoch(), f.run_epoch()
    assert all(math.isfinite(r[k]) for r in (a, b) for k in ("train_loss", "test_loss"))


def test_compiled_model(dev):
    from spotv2net_amd import synthetic_batch
    model, _ = build(dev, hidden=(16, 8))
    data = synthetic_batch(2, 2, seed=1, device=dev)
    want = model(data)
    got = torch.compile(model, backend="aot_eager")(data)
    assert_close(got, want, what="compiled")


def _rank(rank, world, port, out_dir):
    import os
    import torch.distributed as dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    torch.cuda.set_device(0)
    dev = torch.device("cuda", 0)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from spotv2net_amd import synthetic_batch
        from spotv2net_amd.train import TrainStep, broadcast_params_
        model = build(dev, hidden=(16, 8), seed=20 + rank)[0].train()
        broadcast_params_(model, 0)
        data = synthetic_batch(4, 2, seed=70 + rank, device=dev)
        step = TrainStep(model, data, lr=1e-2, use_graph=True, optimizer="muon")
        assert step.distributed and step._shapes[0].g_opt is not None
        for _ in range(3):
            step()
        torch.cuda.synchronize()
        torch.save({k: v.detach().cpu() for k, v in model.state_dict().items()},
                   os.path.join(out_dir, f"rank{rank}.pt"))
    finally:
        dist.destroy_process_group()


def test_two_ranks_stay_identical(dev, tmp_path):
    """Two data-parallel ranks (gloo, sharing the GPU) under Muon: the replicas end bit
    for bit the same, and moved."""
    import socket

    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.start_processes(_rank, args=(2, port, str(tmp_path)), nprocs=2, join=True,
                       start_method="spawn")
    r0, r1 = (torch.load(tmp_path / f"rank{r}.pt", weights_only=True) for r in range(2))
    start = build(torch.device("cpu"), hidden=(16, 8), seed=20)[0].state_dict()
    for k in r0:
        assert torch.equal(r0[k], r1[k]), k
    assert not torch.equal(r0["gat_layers.0.lin_src.weight"], start["gat_layers.0.lin_src.weight"])
