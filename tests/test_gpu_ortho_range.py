"""Orthogonalisation of matrices whose rows and columns differ by many orders of
magnitude, under few and many steps and coefficients that let small parts grow or X
shrink, against the definition in 64 bits.

Allowed (2-norm, relative): three times the error of the same steps in plain f32
products, at least 3e-5, as for ordinary matrices, over the whole matrix at any steps and
coefficients.  The small part by itself, relative to its own norm: the same where the
products are f32; with pairs of f16 an entry may be off by 2^-39 of the whole besides
(2^-41 on average over roundings), multiplied by the steps' largest gain."""
import math

import pytest
import torch

from test_gpu_ortho import HALF, NS, definition, rel

pytestmark = pytest.mark.gpu

FAST = (15 / 8, -10 / 8, 3 / 8)
CUBIC = (1.5, -0.5, 0.0)


def graded(dev, rows, cols, small, where, seed=0):
    """Noise, the second half of the rows, the columns or both times `small`; its part."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    g = torch.randn(rows, cols, device=dev, generator=gen)
    if where == "rows":
        part = (slice(rows // 2, None), slice(None))
        g[part] *= small
    elif where == "cols":
        part = (slice(None), slice(cols // 2, None))
        g[part] *= small
    else:  # a block of its own, orthogonal to the large one
        part = (slice(rows // 2, None), slice(cols // 2, None))
        g[part] *= small
        g[:rows // 2, cols // 2:] = 0
        g[rows // 2:, :cols // 2] = 0
    return g, part


def bound(g, ref, part=(slice(None), slice(None)), **kw):
    return max(3 * rel(definition(g, dtype=torch.float32, **kw)[part], ref[part]), 3e-5) + \
        HALF[g.dtype]


@pytest.mark.parametrize("small", [1e-4, 1e-6, 1e-8, 1e-10, 1e-12])
@pytest.mark.parametrize("where", ["rows", "cols", "block"])
@pytest.mark.parametrize("rows,cols", [(64, 128), (300, 200), (700, 900)])
@pytest.mark.parametrize("steps,co", [(5, NS), (8, NS), (16, NS), (24, NS), (32, FAST), (32, CUBIC)])
def test_whole_matrix(dev, small, where, rows, cols, steps, co):
    from spotv2net_amd import orthogonalize
    g, part = graded(dev, rows, cols, small, where, seed=rows + steps)
    ref = definition(g, steps=steps, co=co)
    u = orthogonalize(g, steps=steps, coefficients=co)
    assert rel(u, ref) <= bound(g, ref, steps=steps, co=co)
    if steps >= 16:  # f32 products
        assert rel(u[part], ref[part]) <= bound(g, ref, part, steps=steps, co=co)
    elif steps == 5:
        room = 3e-5 * float(ref[part].norm()) + \
            2 * NS[0] * 4.0 ** 4 * 2.0 ** -40.8 * math.sqrt(g[part].numel())
        assert float((u[part].double() - ref[part]).norm()) <= room


@pytest.mark.parametrize("rows,cols", [(1, 1), (40, 50), (128, 1024), (1500, 1300), (3, 4000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_many_steps(dev, rows, cols, dtype):
    """Ordinary matrices on the f32 products, every type and tile."""
    from spotv2net_amd import orthogonalize
    gen = torch.Generator(device=dev).manual_seed(rows)
    g = torch.randn(rows, cols, device=dev, generator=gen).to(dtype)
    for steps, co in ((12, NS), (20, FAST)):
        ref = definition(g, steps=steps, co=co)
        assert rel(orthogonalize(g, steps=steps, coefficients=co), ref) <= \
            bound(g, ref, steps=steps, co=co), steps


@pytest.mark.parametrize("co,steps", [((0.5, 0.0, 0.0), 32), ((0.1, 0.0, 0.0), 20),
                                      ((0.3, 0.2, -0.1), 12), ((-0.4, 0.1, 0.0), 15)])
@pytest.mark.parametrize("rows,cols", [(64, 128), (700, 900)])
def test_shrinking_coefficients(dev, co, steps, rows, cols):
    from spotv2net_amd import orthogonalize
    gen = torch.Generator(device=dev).manual_seed(7)
    g = torch.randn(rows, cols, device=dev, generator=gen)
    ref = definition(g, steps=steps, co=co)
    assert rel(orthogonalize(g, steps=steps, coefficients=co), ref) <= \
        bound(g, ref, steps=steps, co=co)


def test_stack(dev):
    from spotv2net_amd import orthogonalize
    g = torch.stack([graded(dev, 130, 260, s, "rows", seed=k)[0]
                     for k, s in enumerate((1.0, 1e-8, 1e-10))])
    u = orthogonalize(g, steps=16)
    for k in range(3):
        ref = definition(g[k], steps=16)
        assert rel(u[k], ref) <= bound(g[k], ref, steps=16), k


@pytest.mark.parametrize("shapes", [[(700, 900), (5, 3000), (900, 31), (32, 32)],
                                    [(64, 128), (20, 60), (8, 8)], [(1500, 1600), (3, 2)]])
def test_optimizer_step(dev, shapes):
    """Large, small and thin matrices of one step under many Newton-Schulz steps."""
    from spotv2net_amd import muon_step
    gs = [graded(dev, m, n, 1e-8, "rows", seed=k)[0] for k, (m, n) in enumerate(shapes)]
    ws, ms = [torch.zeros_like(g) for g in gs], [torch.zeros_like(g) for g in gs]
    muon_step(ws, gs, ms, lr=1.0, momentum=0.0, steps=16)
    for w, g in zip(ws, gs):
        ref = definition(g, steps=16) * -math.sqrt(max(1.0, g.shape[0] / g.shape[1]))
        f32 = rel(definition(g, steps=16, dtype=torch.float32), definition(g, steps=16))
        assert rel(w, ref) <= max(3 * f32, 3e-5), tuple(g.shape)


def test_long_thin_neighbour(dev):
    """A thin matrix is on f32 products anyway: beside it the others keep theirs (the
    bits of the step without it)."""
    from spotv2net_amd import muon_step
    g, t = graded(dev, 96, 128, 1.0, "rows")[0], graded(dev, 30, 16384, 1.0, "rows", seed=1)[0]
    both, alone = [torch.zeros_like(g), torch.zeros_like(t)], [torch.zeros_like(g)]
    for steps in (8, 16):
        muon_step(both, [g, t], [torch.zeros_like(g), torch.zeros_like(t)], lr=1.0, momentum=0.0,
                  steps=steps)
        muon_step(alone, [g], [torch.zeros_like(g)], lr=1.0, momentum=0.0, steps=steps)
        assert torch.equal(both[0], alone[0]), steps
