"""Orthogonalised updates against the products in float64.

Bound.  One step maps singular values by p(s) = a s + b s^3 + c s^5; how much it enlarges a small change of X, in the Frobenius norm, is the
largest of |p(s_i) - p(s_j)| / |s_i - s_j| (p' where they meet), |p(s_i) + p(s_j)| / (s_i + s_j) and |p(s_i)| / s_i, taken here from the singular
values of every step.  A step itself adds what its products are off: every operand by at most `held` of itself, a product's sum by at
most `summed` of its terms' magnitudes, and X by one rounding of float32.  The sum of these, each enlarged by the steps that follow,
bounds the result to first order (a factor 1.5 covers the rest); bfloat16 results are rounded once more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
USUAL = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "the gpu tests need a CUDA device"
    return torch.device("cuda:0")


def gain(s, coefficients):
    a, b, c = coefficients
    p = a * s + b * s ** 3 + c * s ** 5
    d = a + 3 * b * s ** 2 + 5 * c * s ** 4
    near = (s[:, None] - s[None]).abs() < 1e-6
    minus = torch.where(near, d[:, None].expand(len(s), len(s)), (p[:, None] - p[None]) / (s[:, None] - s[None]).masked_fill(near, 1.0))
    total = s[:, None] + s[None]
    plus = torch.where(total < 1e-9, torch.full_like(total, a), (p[:, None] + p[None]) / total.clamp_min(1e-9))
    return max(minus.abs().max().item(), plus.abs().max().item(), d.abs().max().item())


def reference(U, steps, coefficients, eps, dtype):
    """The result of one matrix in float64 and the bound of its distance in the Frobenius norm."""
    a, b, c = coefficients
    X = U.double()
    X = X / (X.norm() + eps)
    if X.shape[0] > X.shape[1]:
        out, bound = reference(U.t(), steps, coefficients, eps, dtype)
        return out.t(), bound
    held = 2.0 ** -22 if dtype == F32 else 2.0 ** -11
    # float32: three terms of 64 k in 12 truncating additions (2^-22), the chunks and the low parts' product beside them
    summed = lambda K: 13 * 2.0 ** -22 + (K / 64 + 1) * 2.0 ** -24 if dtype == F32 else (K / 16 + 1) * 2.0 ** -22  # noqa: E731
    fro = lambda M: M.norm().item()  # noqa: E731
    off = 2 * 2.0 ** -24 * fro(X)
    for _ in range(steps):
        s = torch.linalg.svdvals(X)
        top = s.max().item()
        S = X @ X.t()
        P = b * S + c * S @ S
        eS = (2 * held + summed(X.shape[1])) * fro(X.abs() @ X.abs().t())
        eP = abs(b) * (eS + held * fro(S)) + abs(c) * (2 * top * top * eS + (2 * held + summed(S.shape[0])) * fro(S.abs() @ S.abs()))
        eX = eP * top + (2 * held + summed(S.shape[0])) * fro(P.abs() @ X.abs()) + 4 * 2.0 ** -24 * (abs(a) * fro(X) + fro(P @ X))
        off = off * gain(s, coefficients) + eX
        X = a * X + P @ X
    u = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
    return X, 1.5 * off + u * fro(X)


def update(seed, shape, dtype, dev, kind="normal"):
    g = torch.Generator().manual_seed(seed)
    U = torch.randn(*shape, generator=g, dtype=torch.float64)
    m, n = shape[-2:]
    if kind == "even":      # all singular values within a factor of four
        q = torch.linalg.qr(torch.randn(*shape[:-2], max(m, n), min(m, n), generator=g, dtype=torch.float64))[0]
        U = q * torch.exp(math.log(4) * torch.rand(min(m, n), generator=g, dtype=torch.float64))
        U = U if m >= n else U.transpose(-1, -2)
    elif kind == "low rank":
        r = max(1, min(m, n) // 4)
        U = torch.randn(*shape[:-2], m, r, generator=g, dtype=torch.float64) @ torch.randn(*shape[:-2], r, n, generator=g, dtype=torch.float64)
    return U.to(dtype).to(dev)


def check(out, U, steps=5, coefficients=USUAL, eps=1e-7):
    assert out.shape == U.shape and out.dtype == U.dtype
    assert torch.isfinite(out).all()
    for got, u in zip(out.reshape(-1, *U.shape[-2:]), U.reshape(-1, *U.shape[-2:])):
        want, bound = reference(u, steps, coefficients, eps, U.dtype)
        off = (got.double() - want).norm().item()
        assert off <= bound, f"{off:.2e} off, bound {bound:.2e}"


SHAPES = [(1, 1, 1), (3, 1, 40), (2, 40, 1), (4, 64, 64), (2, 16, 23), (3, 100, 64), (2, 128, 128), (2, 128, 512), (1, 512, 96), (1, 129, 130),
          (1, 130, 129), (2, 250, 70), (1, 257, 640), (3, 5, 200), (1, 600, 300), (40, 140, 300), (40, 300, 140)]


@pytest.mark.parametrize("kind", ["even", "normal", "low rank"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_values(shape, dtype, kind, dev):
    from cuda_mace_b200 import ops

    U = update(sum(shape), shape, dtype, dev, kind)
    check(ops.orthogonalize(U), U)
    ops.check_status()
