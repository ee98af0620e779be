"""Layer norm without a GPU: what the C entries refuse (before any launch), the
module's constructor, and the refusal of CPU tensors."""
import pytest
import torch


def _lib():
    from spotv2net_amd import _lib
    return _lib.load()


FAKE = 1 << 20  # a device address the entry must refuse before using


def _fwd(lib, x=FAKE, ldx=8, dtype=0, w=None, b=None, wdtype=0, rows=4, cols=8, eps=1e-5, y=FAKE):
    return lib.sv2n_layer_norm_fwd(x, ldx, dtype, w, b, wdtype, rows, cols, eps, y, None, None, None)


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), -1), (dict(y=None), -1), (dict(rows=-1), -1), (dict(cols=0), -1),
    (dict(eps=-1e-5), -1), (dict(eps=float("nan")), -1), (dict(dtype=3), -1), (dict(dtype=-1), -1),
    (dict(wdtype=1), -1), (dict(dtype=1, wdtype=2), -1),
    (dict(ldx=7), -2), (dict(cols=16385, ldx=16385), -2),
    (dict(x=FAKE + 2), -3), (dict(y=FAKE + 1), -3), (dict(dtype=1, x=FAKE + 1), -3),
    (dict(rows=0, x=None, y=None), 0)])
def test_forward_refusals(kw, code):
    assert _fwd(_lib(), **kw) == code


def _bwd(lib, dy=FAKE, lddy=8, x=FAKE, ldx=8, dtype=0, wdtype=0, mean=FAKE, rstd=FAKE, rows=4,
         cols=8, dx=FAKE, dw=FAKE, db=FAKE, acc=0, ws=FAKE, ws_n=1 << 40):
    return lib.sv2n_layer_norm_bwd(dy, lddy, x, ldx, dtype, None, wdtype, mean, rstd, rows, cols,
                                   dx, dw, db, acc, ws, ws_n, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dy=None), -1), (dict(x=None), -1), (dict(mean=None), -1), (dict(rstd=None), -1),
    (dict(rows=-1), -1), (dict(cols=0), -1), (dict(wdtype=2), -1), (dict(lddy=7), -2),
    (dict(ldx=7), -2), (dict(cols=16385, ldx=16385, lddy=16385), -2), (dict(dx=FAKE + 2), -3),
    (dict(ws=None), -4), (dict(ws_n=15), -4),
    (dict(dx=None, dw=None, db=None), 0), (dict(rows=0, acc=1), 0),
    (dict(rows=0, dw=None, db=None), 0)])
def test_backward_refusals(kw, code):
    assert _bwd(_lib(), **kw) == code


def test_workspace_covers_the_partials():
    lib = _lib()
    assert lib.sv2n_layer_norm_bwd_workspace(0, 8, 0) == 0
    assert lib.sv2n_layer_norm_bwd_workspace(8, 0, 0) == 0
    assert lib.sv2n_layer_norm_bwd_workspace(8, 16385, 0) == 0
    for rows, cols, dt in ((1, 1, 0), (30, 400, 0), (1 << 20, 128, 1), (7, 16384, 2)):
        n = lib.sv2n_layer_norm_bwd_workspace(rows, cols, dt)
        assert n % (2 * cols) == 0 and 1 <= n // (2 * cols) <= 1024


def test_module_surface():
    from spotv2net_amd import LayerNorm
    m, r = LayerNorm(12, eps=1e-3), torch.nn.LayerNorm(12, eps=1e-3)
    assert list(m.state_dict()) == list(r.state_dict()) and m.eps == 1e-3
    m.load_state_dict(r.state_dict())
    assert list(LayerNorm(12, bias=False).state_dict()) == ["weight"]
    assert not list(LayerNorm(12, elementwise_affine=False).state_dict())
    with pytest.raises(ValueError, match="last dimension"):
        LayerNorm((3, 4))
    with pytest.raises(RuntimeError, match="rows of 5"):
        m(torch.randn(2, 5))


def test_refuses_cpu_tensors():
    from spotv2net_amd import layer_norm
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        layer_norm(torch.randn(3, 4))


def test_refuses_forward_mode():
    import torch.autograd.forward_ad as fw
    import spotv2net_amd  # noqa: F401
    x, w = torch.randn(3, 4), torch.randn(4)
    with fw.dual_level():
        for args in ((fw.make_dual(x, x), w), (x, fw.make_dual(w, w))):
            with pytest.raises(RuntimeError, match="no forward-mode"):
                torch.ops.sv2n.layer_norm(*args, None, 1e-5)


def test_fake_tensors_propagate_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    import spotv2net_amd  # noqa: F401
    with FakeTensorMode():
        x = torch.empty(3, 5, 8, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(8, device="cuda")
        y, mean, rstd = torch.ops.sv2n.layer_norm(x, w, None, 1e-5)
        assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == rstd.shape == (15,)
        dx, dw, db = torch.ops.sv2n.layer_norm_bwd(y, x, w, mean, rstd, True, True, False)
        assert dx.shape == x.shape and dw.shape == (8,) and dw.dtype == torch.float32
        assert db.numel() == 0
