"""What TrainStep and Fit refuse before they touch the model (no GPU)."""
import pytest
import torch


def _model():
    from spotv2net_amd import GATModel
    return GATModel(60, 6, 2, 1, [8, 4], concat_heads=True)


@pytest.mark.parametrize("name", ["Muon", "adam", "sgd", "", "sv2n ", None])
def test_unknown_optimizer(name):
    from spotv2net_amd.train import TrainStep
    model = _model()
    before = [(p.data_ptr(), p.grad) for p in model.parameters()]
    with pytest.raises(ValueError, match="optimizer is"):
        TrainStep(model, None, use_graph=False, optimizer=name)
    assert [(p.data_ptr(), p.grad) for p in model.parameters()] == before


def test_unknown_optimizer_in_the_loop():
    from spotv2net_amd import WindowDataset, synthetic_series
    from spotv2net_amd.train import Fit, fit
    vol, volvol = synthetic_series(20, n=30, seed=1)
    ds = WindowDataset(vol, volvol, 2)
    model = _model()
    model.eval()
    for call in (lambda: Fit(model, ds, 4, optimizer="adamw"),
                 lambda: fit(model, ds, 1, 4, optimizer="adamw")):
        with pytest.raises(ValueError, match="optimizer is"):
            call()
    assert not model.training
    assert all(p.grad is None for p in model.parameters())
    assert isinstance(model.gat_layers[0].lin_src.weight, torch.nn.Parameter)


def test_model_pickled_without_norms():
    """A whole model pickled before it could hold norms is a model without them."""
    import copy
    import io
    model = _model()
    old = copy.deepcopy(model)
    del old.__dict__["norms"]
    buf = io.BytesIO()
    torch.save(old, buf)
    buf.seek(0)
    again = torch.load(buf, weights_only=False)  # (this test's own bytes)
    assert again.norms is None
    assert copy.deepcopy(again).norms is None
    from spotv2net_amd import GATModel
    normed = GATModel(60, 6, 2, 1, [8, 4], concat_heads=True, layer_norm=True)
    assert len(copy.deepcopy(normed).norms) == 2
