"""The gated feed-forward block against its formulas in float64, element by element.

Bounds.  u is half a step of the type.  bfloat16 rounds the hidden values h (and, going back, dL/dg and dL/du) once and the result once,
all by at most u = 2^-8 relative; the sums between are float32.  float32 goes as pairs of fp16 values: an operand is off by at most 2^-22
of itself (and 2^-39 of its block's largest value), the product of the two low parts (2^-22) is left out, and 64 k are summed in 12 truncating
additions of at most 2^-22 of the sum of the magnitudes, then added with rounding (2^-24): `product_bound` adds these up over the sum of
the terms' magnitudes, which no order of summation exceeds."""
import math

import pytest
import torch

from tests.util import rel_err

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "the gpu tests need a CUDA device"
    return torch.device("cuda:0")


def act_of(g, activation):
    """act(g), act'(g), both from the definition."""
    if activation == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def product_bound(A, B, dtype, dA=0.0, dB=0.0):
    """How far a product of A and B as the kernels hold them may be from A @ B, dA and dB being what the operands are off already."""
    K = A.shape[1]
    mag = A.abs() @ B.abs()
    if dtype == F32:
        # blocks of 64 x 64 share a scale: 2^-39 of the largest value of the whole matrix bounds what small values lose
        small = 2.0 ** -39 * (A.abs().max() * B.abs().sum(0) + B.abs().max() * A.abs().sum(1, keepdim=True)) if A.numel() and B.numel() else 0.0
        own = (3 * 2.0 ** -22 + 12 * 2.0 ** -22 + (K / 64 + 64) * 2.0 ** -24) * mag + small
    else:
        own = (K / 16 + 64) * 2.0 ** -22 * mag
    if torch.is_tensor(dA):
        own = own + dA @ (B.abs() + (dB if torch.is_tensor(dB) else 0.0))
    if torch.is_tensor(dB):
        own = own + A.abs() @ dB
    return own


def reference(x, wg, wu, wd, gy, activation, dtype):
    """Values in float64 and the bound of each, for operands that are given in `dtype`."""
    u = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
    held = u if dtype == BF16 else 0.0    # what a hidden value loses when it is put down (float32: the pairs' part of product_bound)
    g, up = x @ wg, x @ wu
    eg, eu = product_bound(x, wg, dtype), product_bound(x, wu, dtype)
    a, da = act_of(g, activation)
    # |act'| <= 1.13 and |act''| <= 0.8 for both; the functions themselves to 16 rounding steps of their size
    ea = 1.13 * eg + 2.0 ** -20 * (a.abs() + 2.0 ** -126) + (2.0 ** -22 * g.abs() if activation == "gelu" else 0.0)
    eda = 0.8 * eg + 2.0 ** -20 * (da.abs() + g.abs() * 2.0 ** -4)
    h = a * up
    eh = ea * (up.abs() + eu) + a.abs() * eu
    eh = eh + held * (h.abs() + eh) + 2.0 ** -23 * h.abs()
    y = h @ wd
    ey = product_bound(h, wd, dtype, dA=eh)
    out = {"y": (y, ey + u * (y.abs() + ey))}
    if gy is None:
        return out
    dh = gy @ wd.t()
    edh = product_bound(gy, wd.t(), dtype)
    dg, du = dh * up * da, dh * a
    edg = (dh.abs() + edh) * (up.abs() + eu) * (da.abs() + eda) - dg.abs()
    edu = (dh.abs() + edh) * (a.abs() + ea) - du.abs()
    edg, edu = (e + held * (v.abs() + e) + 2.0 ** -22 * v.abs() for e, v in ((edg, dg), (edu, du)))
    gx = dg @ wg.t() + du @ wu.t()
    ex = product_bound(dg, wg.t(), dtype, dA=edg) + product_bound(du, wu.t(), dtype, dA=edu)
    out["x"] = (gx, ex + u * (gx.abs() + ex))
    for name, A, B, eB in (("w_gate", x, dg, edg), ("w_up", x, du, edu)):
        v, e = A.t() @ B, product_bound(A.t(), B, dtype, dB=eB)
        out[name] = (v, e + u * (v.abs() + e))
    v, e = h.t() @ gy, product_bound(h.t(), gy, dtype, dA=eh.t())
    out["w_down"] = (v, e + u * (v.abs() + e))
    return out


def case(seed, M, C, H, dtype, dev, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x = r(M, C) * torch.exp(spread * r(M, 1))
    t = [x, r(C, H) / math.sqrt(C), r(C, H) / math.sqrt(C), r(H, C) / math.sqrt(H), r(M, C)]
    return [v.to(dtype).to(dev) for v in t]


def inside(got, want):
    v, bound = want
    off = (got.double() - v).abs()
    assert torch.isfinite(got).all()
    worst = (off / bound.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert (off <= bound + 1e-37).all(), f"{worst:.2f} times the bound"


SIZES = [
    (1, 128, 512), (2, 1, 1), (3, 7, 5), (63, 64, 64), (64, 32, 128), (65, 96, 192), (127, 130, 66), (128, 128, 256), (129, 100, 129),
    (200, 8, 1001), (5, 250, 40), (257, 257, 65), (1000, 128, 512), (300, 512, 130),
    (20001, 40, 136), (9999, 264, 300),   # enough rows for pairs of CTAs, 128 and 256 columns a tile
]


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,C,H", SIZES)
def test_forward(M, C, H, dtype, activation, dev):
    from cuda_mace_b200 import ops

    x, wg, wu, wd, _ = case(M + C + H, M, C, H, dtype, dev)
    y = ops.gated_feed_forward(x, wg, wu, wd, activation=activation)
    assert y.shape == x.shape and y.dtype == dtype
    inside(y, reference(*(t.double() for t in (x, wg, wu, wd)), None, activation, dtype)["y"])
    ops.check_status()


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,C,H", SIZES + [(5000, 32, 64), (20000, 16, 24)])
def test_gradients(M, C, H, dtype, activation, dev):
    from cuda_mace_b200 import ops

    x, wg, wu, wd, gy = case(M + C + H + 1, M, C, H, dtype, dev)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = ops.gated_feed_forward(*leaves, activation=activation)
    grads = torch.autograd.grad(y, leaves, gy)
    want = reference(*(t.double() for t in (x, wg, wu, wd, gy)), activation, dtype)
    for name, got in zip(("x", "w_gate", "w_up", "w_down"), grads):
        assert got.dtype == dtype
        inside(got, want[name])
    ops.check_status()
