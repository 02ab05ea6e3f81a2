"""GELU where its gate is nearly closed: values against their own size, not against the activation's largest.

One channel of x is the argument v, another is one, and the weights pass them on, so that y is gelu(v) in every column.  What v is off by,
3 * 2^-22 of it (a pair, the truncation that is put back), changes v cdf(v) by (1 + v^2) of that in the tail; the exponential of -z^2 = -v^2 / 2 is off
by 2^-22 (1 + z^2), the fit by 2e-6 up to z = 4, the products and pairs behind it by 2^-20: together below 2^-18 (1 + z^2)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def gelu(v):
    """Value and derivative."""
    cdf, pdf = 0.5 * torch.special.erfc(-v / math.sqrt(2)), torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    return v * cdf, cdf + v * pdf, cdf + v.abs() * pdf


@pytest.mark.parametrize("low,high", [(-6.0, -5.0), (-5.0, -4.0), (-4.0, -3.0), (-3.0, -2.0), (-2.0, 0.0), (0.0, 6.0)])
@pytest.mark.parametrize("M,C,H", [(5, 160, 1030), (60, 64, 64), (300, 136, 200)])   # few rows, some rows, tiles
def test_tail(M, C, H, low, high):
    from cuda_mace_b200 import ops

    v = torch.linspace(low, high, M + 2, dtype=torch.float64)[1:-1].float().cuda()
    x = torch.zeros(M, C, device="cuda")
    x[:, 0], x[:, 1] = v, 1
    wg, wu, wd = torch.zeros(C, H, device="cuda"), torch.zeros(C, H, device="cuda"), torch.zeros(H, C, device="cuda")
    wg[0], wu[1] = 1, 1
    k = torch.arange(min(C, H), device="cuda")
    wd[k, k] = 1
    leaf = x.requires_grad_(True)
    y = ops.gated_feed_forward(leaf, wg, wu, wd, activation="gelu")
    value, slope, size = (t[:, None] for t in gelu(v.double()))
    tolerance = 2.0 ** -18 * (1 + v.double()[:, None] ** 2 / 2)
    got = y.detach().double()[:, :len(k)]
    assert ((got - value).abs() <= tolerance * value.abs()).all(), ((got - value).abs() / value.abs() / tolerance).max()
    # the slope, by a gradient of one column: against its two terms, which cancel nowhere by more than v^2
    gy = torch.zeros(M, C, device="cuda")
    gy[:, 0] = 1
    (g,) = torch.autograd.grad(y, leaf, gy)
    off = (g[:, :1].double() - slope).abs()
    assert (off <= tolerance * size).all(), (off / size / tolerance).max()
