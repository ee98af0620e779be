"""What 16-bit results of the orthogonalisation keep: nothing is lost beside the one
rounding of the result, whatever part of the matrix is filled.

A result is the exact one, off by an f32 error d (2-norm at most 3e-5 of the result's:
five steps of about 8 roundings of 2^-22 to 2^-24, each handed on at most doubled), then
rounded.  Rounding a value that is off by d gives what rounding the exact one gives, or
its neighbour where the exact one lies within d of the middle between them: further off by
2 d at most.  So the result may be off by what rounding the exact one costs plus 6e-5."""
import pytest
import torch

from test_gpu_ortho import definition, rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n", [(128, 300), (300, 128), (200, 3000), (1024, 1100)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 2), (4, 8), (16, 16), (1, None), (16, None),
                                       (None, 3), (None, None)])
def test_rounded_once(dev, dtype, m, n, rows, cols):
    """A block of `rows` x `cols` filled (None: all of them), zeros elsewhere."""
    from spotv2net_amd import orthogonalize
    gen = torch.Generator(device=dev).manual_seed(m + n)
    g = torch.zeros(m, n, device=dev)
    g[:rows, :cols] = torch.randn(rows or m, cols or n, device=dev, generator=gen)
    g = g.to(dtype)
    ref = definition(g)
    assert rel(orthogonalize(g), ref) <= rel(ref.to(dtype), ref) + 6e-5


def test_low_rank_of_one_sign(dev):
    """Roundings that all go the same way: constant matrices and outer products."""
    from spotv2net_amd import orthogonalize
    gen = torch.Generator(device=dev).manual_seed(5)
    for m, n in ((128, 128), (1024, 1500)):
        u = torch.rand(m, 1, device=dev, generator=gen) + 0.5
        v = torch.rand(1, n, device=dev, generator=gen) + 0.5
        for g in (torch.full((m, n), 0.7, device=dev), u * v, u.expand(m, n)):
            g = g.bfloat16()
            ref = definition(g)
            assert rel(orthogonalize(g), ref) <= rel(ref.bfloat16(), ref) + 6e-5, (m, n)
