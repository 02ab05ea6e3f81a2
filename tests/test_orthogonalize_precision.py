"""bfloat16 updates against the rounding of their own result.

The general bound of an update multiplies every step's rounding by the worst gain of all singular values, which in bfloat16 allows more than the
result's size.  On updates whose singular values lie within a factor of four there is a sharper measure: the error of the result, as a norm,
over that of rounding the exact result to bfloat16.  The kernels' own rounding points, emulated here in float64 (X, S and P as pairs of fp16
values), come to 1.0 of it where every product has three terms (shorter side up to 128, longer up to 1024) and to 1.33 to 1.49 where products but S S take the high
values alone; bfloat16 operands throughout to 6 and more.  The limits are these and a tenth of the rounding for float32 sums and
truncating additions, which are off by less than 2^-12 a product: in squares (2^-12 / 2^-9)^2 = 1/64 each, 15 products, and less along what grows."""
import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16
A, B, C = 3.4445, -4.7750, 2.0315


def even(seed, count, m, n):
    """Singular values within a factor of four, bfloat16."""
    g = torch.Generator().manual_seed(seed)
    q = torch.linalg.qr(torch.randn(count, max(m, n), min(m, n), generator=g, dtype=torch.float64))[0]
    v = torch.linalg.qr(torch.randn(count, min(m, n), min(m, n), generator=g, dtype=torch.float64))[0]
    U = (q * torch.exp(1.386 * torch.rand(min(m, n), generator=g, dtype=torch.float64))) @ v
    return (U if m >= n else U.transpose(-1, -2)).to(BF16)


def start(U):
    X = U.double()
    X = X / (X.norm(dim=(-2, -1), keepdim=True) + 1e-7)
    return X.transpose(-1, -2) if X.shape[-2] > X.shape[-1] else X


def products(U, steps=5):
    X = start(U)
    for _ in range(steps):
        S = X @ X.transpose(-1, -2)
        X = A * X + (B * S + C * S @ S) @ X
    return X


def pair(x, most):
    """High and low part of x as fp16 values at a power of two that keeps values up to `most` below 2^15."""
    scale = 2.0 ** 15 / 2.0 ** torch.ceil(torch.log2(torch.tensor(1.05 * most, dtype=torch.float64))).item()
    hi = (x * scale).half().double()
    lo = (x * scale - hi).half().double()
    return hi / scale, lo / scale


def emulated(U, all_terms):
    """The kernels' rounding points; all_terms: of updates whose shorter side is up to 128, which take three terms in every product."""
    X, most = start(U), 1.0
    for _ in range(5):
        h, l = pair(X, most)
        S = h @ h.transpose(-1, -2) + ((h @ l.transpose(-1, -2) + l @ h.transpose(-1, -2)) if all_terms else 0.0)
        sh, sl = pair(S, most * most)
        P = B * (sh + sl) + C * (sh @ sh + sh @ sl + sl @ sh)
        t = torch.linspace(0, most, 10001, dtype=torch.float64)
        ph, pl = pair(P, (t * t * (B + C * t * t)).abs().max().item())
        X = A * (X if all_terms else h + l) + ph @ h + ((ph @ l + pl @ h) if all_terms else 0.0)
        most = (t * (A + t * t * (B + t * t * C))).abs().max().item()
    return X.to(BF16)


def in_bfloat16(U):
    r = lambda x: x.to(BF16).double()  # noqa: E731
    X = r(start(U))
    for _ in range(5):
        S = r(X @ X.transpose(-1, -2))
        X = r(A * X + r(B * S + C * S @ S) @ X)
    return X.to(BF16)


def times_rounding(got, want):
    """The largest error of a matrix, as a norm, over that of the exact result's rounding."""
    err = lambda x: (x.double() - want).norm(dim=(-2, -1))  # noqa: E731
    return (err(got) / err(want.to(BF16))).max().item()


def limit(shape):
    return 1.1 if min(shape[1:]) <= 128 else 1.65


SIDES = [(4, 64, 64), (2, 128, 512), (2, 512, 96), (1, 257, 640), (1, 600, 300), (2, 140, 300), (1, 512, 1024)]


@pytest.mark.parametrize("shape", SIDES)
def test_the_measure(shape):
    """Accepts the kernels' rounding; rejects zeros, a step left out and bfloat16 operands."""
    U = even(sum(shape), *shape)
    want = products(U)
    assert times_rounding(emulated(U, min(shape[1:]) <= 128), want) <= limit(shape) - 0.05
    for wrong in (torch.zeros_like(want), products(U, 4), products(U, 6), in_bfloat16(U), 3 * want):
        assert times_rounding(wrong, want) > 2 * limit(shape)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SIDES + [(2, 1024, 2048)])
def test_against_its_rounding(shape):
    from cuda_mace_b200 import ops

    U = even(sum(shape), *shape).cuda()
    out = ops.orthogonalize(U)
    out = out.transpose(-1, -2) if shape[1] > shape[2] else out
    assert times_rounding(out, products(U)) <= limit(shape)
