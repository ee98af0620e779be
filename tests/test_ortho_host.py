"""Orthogonalised updates without a GPU: what the C entries refuse before any
launch, the workspace sizes, the optimiser's constructor, CPU tensors refused."""
import ctypes
import math

import pytest
import torch

NS = (3.4445, -4.7750, 2.0315)
FAKE = 1 << 20  # a device address the entry must refuse before using


def _lib():
    from spotv2net_amd import _lib
    return _lib


def _ortho(g=FAKE, ld=8, bs=0, dtype=0, batch=1, rows=4, cols=8, steps=5, co=NS, eps=1e-7, out=FAKE,
           ws=FAKE, ws_n=1 << 60):
    return _lib().load().sv2n_orthogonalize(g, ld, bs, dtype, batch, rows, cols, steps, *co, eps,
                                            out, ws, ws_n, None)


@pytest.mark.parametrize("kw,code", [
    (dict(g=None), -1), (dict(out=None), -1), (dict(dtype=3), -1), (dict(steps=0), -1),
    (dict(steps=33), -1), (dict(eps=0.0), -1), (dict(eps=float("nan")), -1),
    (dict(co=(float("inf"), 0, 0)), -1), (dict(co=(1, float("nan"), 0)), -1),
    (dict(co=(8.0, 0.0, 0.0)), -1),          # 8^5 > 256: the values grow without bound
    (dict(co=(1.0, 0.0, 300.0)), -1),
    (dict(rows=0), -2), (dict(cols=0), -2), (dict(batch=0), -2), (dict(rows=16385), -2),
    (dict(cols=16385, ld=16385), -2), (dict(batch=1025), -2), (dict(ld=7), -2), (dict(bs=-8), -2),
    (dict(g=FAKE + 2), -3), (dict(out=FAKE + 1, dtype=1), -3), (dict(ws=FAKE + 16), -3),
    (dict(ws=None), -4), (dict(ws_n=100), -4)])
def test_orthogonalize_refusals(kw, code):
    assert _ortho(**kw) == code


def _muon(mats, count=None, lr=0.02, beta=0.95, wd=0.1, steps=5, co=NS, eps=1e-7, ws=FAKE,
          ws_n=1 << 60):
    L = _lib()
    arr = (L.MuonMatrix * max(len(mats), 1))(*[L.MuonMatrix(*m) for m in mats])
    return L.load().sv2n_muon_step(ctypes.addressof(arr), len(mats) if count is None else count, lr,
                                   beta, 1, wd, steps, *co, eps, ws, ws_n, None)


GOOD = (FAKE, 2 * FAKE, 3 * FAKE, 8, 8, 1.0)


@pytest.mark.parametrize("mats,kw,code", [
    ([], {}, 0), ([GOOD], dict(count=-1), -1), ([(None,) + GOOD[1:]], {}, -1),
    ([GOOD[:1] + (None,) + GOOD[2:]], {}, -1), ([GOOD[:2] + (None,) + GOOD[3:]], {}, -1),
    ([GOOD[:5] + (float("nan"),)], {}, -1), ([GOOD], dict(beta=1.0), -1),
    ([GOOD], dict(beta=-0.1), -1), ([GOOD], dict(lr=float("nan")), -1),
    ([GOOD], dict(wd=float("inf")), -1), ([GOOD], dict(steps=0), -1), ([GOOD], dict(eps=-1.0), -1),
    ([GOOD], dict(co=(9.0, 0.0, 0.0)), -1), ([GOOD, GOOD[:3] + (0, 8, 1.0)], {}, -2),
    ([GOOD[:3] + (8, 16385, 1.0)], {}, -2), ([(FAKE + 2,) + GOOD[1:]], {}, -3),
    ([GOOD], dict(ws=FAKE + 128), -3), ([GOOD], dict(ws=None), -4), ([GOOD], dict(ws_n=64), -4)])
def test_muon_refusals(mats, kw, code):
    assert _muon(mats, **kw) == code


def test_workspace():
    lib = _lib().load()
    assert lib.sv2n_orthogonalize_workspace(1, 0, 8) == 0
    assert lib.sv2n_orthogonalize_workspace(1, 8, 16385) == 0
    for b, m, n in ((1, 1, 1), (2, 4096, 20)):
        # thin matrices: 32 rows of f32 and two partial S per 128 columns
        w = -(-max(m, n) // 128)
        assert b * w * (32 * 128 + 2 * 1024) * 4 <= lib.sv2n_orthogonalize_workspace(b, m, n) <= \
            b * w * (32 * 128 + 2 * 1024) * 4 + b * 1024 * 8 + 4 * 256
    for b, m, n in ((1, 33, 33), (3, 1537, 777), (1, 128, 1024), (6, 2048, 2048)):
        lo, hi = min(m, n), max(m, n)
        # X, its two transposes, S and Q at 4 B, padded to at most 128 a side
        least = b * 4 * (3 * lo * hi + 2 * lo * lo)
        most = b * 4 * (3 * (lo + 127) * (hi + 127) + 2 * (lo + 127) ** 2) + b * 1024 * 8 + 6 * 256
        assert least <= lib.sv2n_orthogonalize_workspace(b, m, n) <= most
        assert lib.sv2n_orthogonalize_workspace(b, m, n) == lib.sv2n_orthogonalize_workspace(b, n, m) \
            or m != n


def test_common_coefficients_are_taken():
    """Stable polynomials pass the growth check (the refusal that follows is the
    missing workspace's)."""
    for co, steps in ((NS, 5), (NS, 32), ((1.5, -0.5, 0.0), 32), ((15 / 8, -10 / 8, 3 / 8), 12),
                      ((1.0, 0.0, 0.0), 5), ((0.0, 0.0, 0.0), 1), ((2.0, -1.5, 0.5), 8)):
        assert _ortho(co=co, steps=steps, ws=None) == -4, co


def test_learning_rate_scale():
    from spotv2net_amd.muon import lr_scale
    assert lr_scale(100, 400) == 1.0 and lr_scale(400, 100) == 2.0
    assert math.isclose(lr_scale(100, 400, "match_rms_adamw"), 4.0)
    with pytest.raises(ValueError, match="adjust_lr"):
        lr_scale(1, 1, "none")


def test_optimizer_surface():
    from spotv2net_amd import Muon
    w = torch.nn.Parameter(torch.randn(4, 6))
    o = Muon([w], lr=0.1)
    assert o.defaults["lr"] == 0.1 and o.defaults["nesterov"]
    o.step()  # nothing has a gradient
    for bad in (torch.randn(4), torch.randn(2, 3, 4), torch.randn(4, 6).double()):
        with pytest.raises(ValueError, match="2-D float32"):
            Muon([torch.nn.Parameter(bad)])
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(adjust_lr="x")):
        with pytest.raises(ValueError):
            Muon([w], **kw)
    w.grad = torch.randn(4, 6)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        o.step()


def test_refuses_cpu_tensors():
    from spotv2net_amd import muon_step, orthogonalize
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        orthogonalize(torch.randn(3, 4))
    w = torch.randn(3, 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        muon_step([w], [w.clone()], [w.clone()], lr=0.1)


def test_overlap_rule():
    """The spans check behind the operator's refusal, on CPU tensors."""
    from spotv2net_amd.library import _muon_disjoint
    a = torch.zeros(100)
    g = torch.zeros(10)
    w, m, w2, m2 = a[:10], a[10:20], a[20:30], a[30:40]
    assert _muon_disjoint([(w, g, m)])
    assert _muon_disjoint([(w, g, m), (w2, g, m2)])            # shared gradient: only read
    assert not _muon_disjoint([(w, g, m), (w, g, m2)])         # one weight twice
    assert not _muon_disjoint([(w, g, m), (w2, g, m)])         # one momentum twice
    assert not _muon_disjoint([(w, w, m)])                     # the weight as its gradient
    assert not _muon_disjoint([(w, g, w)])
    assert not _muon_disjoint([(a[:10], g, a[9:19])])          # one element
    assert not _muon_disjoint([(w, g, m), (w2, a[25:35], a[50:60])])


def test_fake_tensors_propagate_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    import spotv2net_amd  # noqa: F401
    with FakeTensorMode():
        g = torch.empty(3, 5, 8, device="cuda", dtype=torch.bfloat16)
        u = torch.ops.sv2n.orthogonalize(g, 5, *NS, 1e-7)
        assert u.shape == g.shape and u.dtype == g.dtype
