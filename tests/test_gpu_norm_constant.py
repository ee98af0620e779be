"""Rows whose values are all alike, and rows far from zero beside their spread: the mean
is that of the values, to the last bit where they are alike.

The mean is corrected by the mean of the deviations from it.  Where all are alike the
deviations are a few units in the last place, equal and exact, so is their sum
(n k < 2^24 units), and the corrected mean is the value itself: z = 0, y = bias, and the
variance is 0.  Otherwise the mean is off by the rounding of the last addition, u of its
size (u = 2^-24), and by 30u of the mean deviation from the first mean, which is the
spread and 30u of the size.  A row of more than 1,024 values lies in several waves:
each one's mean is rounded like that, at most u of the size, their weighted mean is off
by no more than that, and the addition that joins them rounds once more: 2u."""
import pytest
import torch

import spotv2net_amd  # noqa: F401

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
COLS = [1, 2, 3, 5, 7, 13, 14, 64, 126, 400, 777, 1000, 1029, 2050, 3000, 4099, 8200, 16381, 16384]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_constant_rows(dev, cols, dtype):
    vals = [1000.0, 30000.0, 0.1, 1000.1, -7e-5, 3.25, -123.456, 1.0 / 3.0]
    if dtype != torch.float16:
        vals += [1e30, -2.7e-30, 16777215.0]
    v = torch.tensor(vals, device=dev).to(dtype)
    x = v[:, None].expand(-1, cols).contiguous()
    gen = torch.Generator(device=dev).manual_seed(cols)
    w = torch.randn(cols, device=dev, generator=gen)
    b = torch.randn(cols, device=dev, generator=gen)
    y, mean, rstd = torch.ops.sv2n.layer_norm(x, w, b, 1e-5)
    assert torch.equal(mean, v.float())
    assert torch.equal(y, b.to(dtype).expand_as(y))
    # (1e-5 rounded to f32, its root and the reciprocal: half a step each)
    assert ((rstd.double() * 1e-5 ** 0.5 - 1).abs() <= 2.5 * U).all()
    y, _, _ = torch.ops.sv2n.layer_norm(x, None, None, 1e-5)
    assert not y.any()


@pytest.mark.parametrize("cols", [7, 126, 500, 1000, 3000, 16384])
@pytest.mark.parametrize("offset", [1e3, 3e4, 1e6])
def test_far_from_zero(dev, cols, offset):
    gen = torch.Generator(device=dev).manual_seed(cols)
    x = torch.randn(64, cols, device=dev, generator=gen) + \
        offset * (1 + torch.rand(64, 1, device=dev, generator=gen))
    y, mean, rstd = torch.ops.sv2n.layer_norm(x, None, None, 1e-5)
    xd = x.double()
    m = xd.mean(1, keepdim=True)
    d = xd - m
    r = 1 / torch.sqrt(d.square().mean(1, keepdim=True) + 1e-5)
    big = xd.abs().amax(1, keepdim=True)
    spread = d.abs().mean(1, keepdim=True)
    em = (1 if cols <= 1024 else 2) * U * big + 30 * U * (spread + 30 * U * big)
    assert ((mean.double()[:, None] - m).abs() <= em).all()
    # of rstd, relative: 32u of its sums, and what the shifted mean adds to the variance
    er = 32 * U + (r * em) ** 2
    z = d * r
    assert ((y.double() - z).abs() <= r * em + (er + 4 * U) * z.abs()).all()
