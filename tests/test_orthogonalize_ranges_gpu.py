"""Orthogonalised updates whose values leave the middle of float32's range on the way."""
import pytest
import torch

from tests.test_orthogonalize_gpu import USUAL, check, update

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "the gpu tests need a CUDA device"
    return torch.device("cuda:0")


def products(U, steps, coefficients, eps):
    a, b, c = coefficients
    X = U.double()
    X = X / (X.norm(dim=(-2, -1), keepdim=True) + eps)
    tall = X.shape[-2] > X.shape[-1]
    X = X.transpose(-1, -2) if tall else X
    for _ in range(steps):
        S = X @ X.transpose(-1, -2)
        X = a * X + (b * S + c * S @ S) @ X
    return X.transpose(-1, -2) if tall else X


def relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


SHAPES = [(2, 48, 80), (2, 30, 700), (1, 200, 150), (1, 300, 130)]   # one CTA, a cluster, a kernel a product


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("steps,coefficients", [(60, (0.5, 0.0, 0.0)), (20, (0.1, 0.0, 0.0)), (100, (0.5, 0.0, 0.0)), (40, (0.25, -0.125, 0.0625)),
                                                (30, (-0.3, 0.1, 0.01)), (3, (1e-9, 1e-10, 1e-11)), (1, (0.0, 1e-30, 0.0)), (1, (0.0, 0.0, 1e-25))])
def test_coefficients_that_shrink(shape, steps, coefficients, dtype, dev):
    """A step's rounding is at most 2^-22 of X as a pair, and as much of the terms that it adds (at most a X here, but for the last two cases, whose
    single product of three operands is off by 2^-19 at most); bfloat16's operands of those are off by 2^-11 each."""
    from cuda_mace_b200 import ops

    U = update(31 + steps, shape, dtype, dev, "even")
    got = ops.orthogonalize(U, steps=steps, coefficients=coefficients)
    want = products(U, steps, coefficients, 1e-7)
    assert torch.isfinite(got).all()
    if want.abs().max() < 1e-36:   # (1e-9)^3 stays, 0.1^40 would not
        return
    a = abs(coefficients[0])
    terms = max(abs(coefficients[1]), abs(coefficients[2])) / a if a else 1.0
    bound = (steps + 4) * 2.0 ** -21 + (2.0 ** -19 if dtype == F32 else 5 * 2.0 ** -11 * min(1.0, 2 * terms)) + (2.0 ** -8 if dtype == BF16 else 0.0)
    assert relative(got, want) <= bound
    ops.check_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_coefficients_that_grow(shape, dtype, dev):
    """Up to the 1e12 that is accepted."""
    from cuda_mace_b200 import ops

    U = update(41, shape, dtype, dev, "even")
    for steps, coefficients in ((11, (12.0, 0.0, 0.0)), (5, (200.0, 0.0, 0.0))):
        got = ops.orthogonalize(U, steps=steps, coefficients=coefficients)
        want = products(U, steps, coefficients, 1e-7)
        assert relative(got, want) <= (steps + 4) * 2.0 ** -21 + 2.0 ** -19 + (2.0 ** -8 if dtype == BF16 else 0.0), (steps, coefficients)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", SHAPES)
def test_usual_coefficients_of_many_steps(shape, dtype, dev):
    from cuda_mace_b200 import ops

    U = update(43, shape, dtype, dev, "even")
    check(ops.orthogonalize(U, steps=12), U, steps=12, coefficients=USUAL)


@pytest.mark.parametrize("ratio", [0.3, 1e-1, 1e-3, 1e-6, 1e-9, 1e-15, 1e-25])
@pytest.mark.parametrize("steps", [1, 5, 9])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(3, 48, 80), (3, 200, 150), (3, 130, 300)])
def test_updates_far_below_eps(shape, dtype, steps, ratio, dev):
    """Norms at `ratio` of eps, so that X begins at `ratio`, beside matrices that are not small.  float32: the bound of the products' rounding,
    which is relative to X.  bfloat16: its rounding of the result, once, and twice that for the products, whose rounding is 2^-3 of it."""
    from cuda_mace_b200 import ops

    U = update(51, shape, F32, dev, "even").double()
    U[1] *= ratio * 1e-7 / U[1].norm()
    U = U.to(dtype)
    out = ops.orthogonalize(U, steps=steps)
    want = products(U, steps, USUAL, 1e-7)
    if dtype == F32:
        check(out, U, steps=steps)
    for got, w in zip(out, want):
        assert torch.isfinite(got).all() and relative(got, w) <= (2.0 ** -8 * 3 if dtype == BF16 else 2.0 ** -16)
    assert torch.equal(out[0], ops.orthogonalize(U[:1], steps=steps)[0]) or shape[1] > 128


@pytest.mark.parametrize("shape", [(2, 48, 80), (2, 200, 150)])
def test_large_eps(shape, dev):
    from cuda_mace_b200 import ops

    U = update(53, shape, F32, dev)
    for eps in (1e3, 1e12, 1e30):
        check(ops.orthogonalize(U, eps=eps), U, eps=eps)


@pytest.mark.parametrize("which", ["rows", "columns"])
@pytest.mark.parametrize("least", [1e-3, 1e-6])
@pytest.mark.parametrize("shape", [(2, 48, 80), (2, 30, 700), (1, 200, 300), (1, 300, 130), (1, 140, 1030)])
def test_rows_and_columns_that_are_small(shape, least, which, dev):
    """float32 updates some of whose rows (columns) are `least` of others, against their own size.  Everything that a step adds to such a row goes with the
    row itself, as does what it is off by: operands 2^-22 and sums 2^-21 of |P| |X| <= 9 a row, five steps of each, on what grows by 3.4 a
    step: below 5 * 9 / 3.4 * 2^-20 = 2^-16 of the row."""
    from cuda_mace_b200 import ops

    U = update(61, shape, F32, dev).double()
    m, n = shape[1:]
    k = m if which == "rows" else n
    f = least ** ((torch.arange(k, device=dev, dtype=torch.float64) * 7 % 10) / 9)
    U = (U * (f[:, None] if which == "rows" else f)).float()
    out, want = ops.orthogonalize(U).double(), products(U, 5, USUAL, 1e-7)
    dim = -1 if which == "rows" else -2
    error = (out - want).norm(dim=dim) / want.norm(dim=dim)
    assert (error <= 2.0 ** -16).all(), error.max().item()
