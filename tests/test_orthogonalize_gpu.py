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


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(2, 48, 80), (1, 200, 150)])
@pytest.mark.parametrize("steps,coefficients,eps", [(1, USUAL, 1e-7), (3, (2.0, -1.5, 0.5), 0.0), (8, (1.5, -0.5, 0.0), 1e-3), (2, (0.0, 1.0, 0.0), 1e-7),
                                                    (2, (1.0, 0.0, 0.0), 1e-7)])
def test_coefficients(shape, steps, coefficients, eps, dtype, dev):
    from cuda_mace_b200 import ops

    U = update(5, shape, dtype, dev)
    check(ops.orthogonalize(U, steps=steps, coefficients=coefficients, eps=eps), U, steps, coefficients, eps)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(3, 40, 56), (3, 200, 150), (2, 30, 700)])
def test_zeros_and_what_is_not_finite(shape, dtype, dev):
    """A matrix of zeros stays one; an infinity or a NaN spoils its own matrix."""
    from cuda_mace_b200 import ops

    U = update(6, shape, dtype, dev)
    want = ops.orthogonalize(U)
    for bad in (0.0, float("inf"), float("nan")):
        V = U.clone()
        if bad == 0.0:
            V[1] = 0
        else:
            V[1, 3, 5] = bad
        out = ops.orthogonalize(V)
        assert torch.equal(out[0], want[0]) and (len(U) < 3 or torch.equal(out[2], want[2]))
        assert not out[1].any() if bad == 0.0 else not torch.isfinite(out[1]).all()


@pytest.mark.parametrize("shape", [(2, 33, 90), (1, 150, 200)])
@pytest.mark.parametrize("size", [1e-25, 1e-12, 1e9, 1e25])
def test_sizes_of_updates(shape, size, dev):
    """With eps = 0 the result does not depend on the update's size."""
    from cuda_mace_b200 import ops

    U = update(7, shape, F32, dev)
    V = U * size
    check(ops.orthogonalize(V, eps=0.0), V, eps=0.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(2, 3, 40, 56), (2, 2, 150, 200)])
def test_layouts(shape, dtype, dev):
    """Stacks of stacks (ElementalLinear's [Z, 4, K, N]), transposed and odd addresses, single matrices, empty stacks."""
    from cuda_mace_b200 import ops

    U = update(8, shape, dtype, dev)
    want = ops.orthogonalize(U)
    assert want.shape == U.shape
    assert torch.equal(ops.orthogonalize(U.view(-1, *shape[-2:])), want.view(-1, *shape[-2:]))
    assert torch.equal(ops.orthogonalize(U[1, 1]), want[1, 1])
    assert torch.equal(ops.orthogonalize(U.transpose(-1, -2).contiguous().transpose(-1, -2)), want)
    room = torch.zeros(U.numel() + 1, dtype=dtype, device=dev)
    room[1:].copy_(U.reshape(-1))
    check(ops.orthogonalize(room[1:].view(shape)), U)
    assert ops.orthogonalize(U[:0]).shape == (0, *shape[1:])
    t = ops.orthogonalize(U.transpose(-1, -2))
    check(t, U.transpose(-1, -2))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(5, 64, 64), (2, 100, 500), (1, 200, 300)])
def test_same_bits_streams_and_graphs(shape, dtype, dev):
    from cuda_mace_b200 import ops

    sets = [update(20 + k, shape, dtype, dev) for k in range(3)]
    want = [ops.orthogonalize(U) for U in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got.append(ops.orthogonalize(sets[k]))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    static = sets[0].clone()
    graphs, outs, pool = [], [], None
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(ops.orthogonalize(static))
        pool = g.pool()
        graphs.append(g)
    for k in (1, 2, 0):
        static.copy_(sets[k])
        for g, out in zip(graphs, outs):
            g.replay()
            assert torch.equal(out, want[k])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(2, 50, 60), (1, 150, 260), (2, 40, 600)])
def test_in_place(shape, dtype, dev):
    """The C entry takes its input as its output."""
    from cuda_mace_b200 import _abi, ops

    U = update(9, shape, dtype, dev)
    want = ops.orthogonalize(U)
    f32 = dtype == F32
    n = _abi.call("cmace_orthogonalize_workspace_bytes", f32, *shape)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _abi.call("cmace_orthogonalize_" + ("f32" if f32 else "bf16"), U.data_ptr(), *shape, 5, *USUAL, 1e-7, U.data_ptr(), ws.data_ptr(), n, 0,
              torch.cuda.current_stream().cuda_stream)
    assert torch.equal(U, want)


def test_refusals_on_the_device(dev):
    from cuda_mace_b200 import _abi, ops

    U = update(10, (2, 20, 30), F32, dev)
    with pytest.raises(RuntimeError, match="may grow"):
        ops.orthogonalize(U, steps=20, coefficients=(10.0, 0.0, 0.0))
    with pytest.raises(RuntimeError, match="bad sizes"):
        ops.orthogonalize(U, steps=0)
    with pytest.raises(RuntimeError, match="bad coefficients"):
        ops.orthogonalize(U, coefficients=(float("nan"), 0.0, 0.0))
    with pytest.raises(RuntimeError, match="bad coefficients"):
        ops.orthogonalize(U, eps=-1.0)
    with pytest.raises(TypeError):
        ops.orthogonalize(U.double())
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.orthogonalize(U.clone().requires_grad_(True))
    with torch.no_grad():
        ops.orthogonalize(U.clone().requires_grad_(True))
    out = torch.full_like(U, 3.0)
    V = update(10, (2, 200, 300), F32, dev)
    with pytest.raises(RuntimeError, match="needed"):
        _abi.call("cmace_orthogonalize_f32", V.data_ptr(), 2, 200, 300, 5, *USUAL, 1e-7, out.data_ptr(), V.data_ptr() & ~255, 16, 0, 0)
    torch.cuda.synchronize()
    assert (out == 3.0).all()


@pytest.mark.parametrize("shape", [(2, 33, 90), (1, 150, 200)])
@pytest.mark.parametrize("size", [1e-40, 1e-35, 1e37])
def test_ends_of_float32(shape, size, dev):
    """Updates whose norm, or its inverse, is no float32 value (1e-40: the update's own values are subnormal)."""
    from cuda_mace_b200 import ops

    V = update(11, shape, F32, dev) * size
    assert torch.isfinite(V).all()
    check(ops.orthogonalize(V, eps=0.0), V, eps=0.0)


def test_long_sides_and_forward_mode_are_refused(dev):
    from torch.autograd import forward_ad

    from cuda_mace_b200 import ops

    with pytest.raises(RuntimeError, match="sides up to"):
        ops.orthogonalize(torch.ones(1, 1, device=dev).expand(1, 2 ** 32 + 16))
    with pytest.raises(RuntimeError, match="bad sizes"):
        ops.orthogonalize(torch.ones(2, 2, device=dev), steps=2 ** 32 + 5)
    U = update(12, (4, 5), F32, dev)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            ops.orthogonalize(forward_ad.make_dual(U, torch.ones_like(U)))
        ops.orthogonalize(U)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(2, 40, 520), (1, 520, 128), (2, 100, 193), (80, 20, 250), (1, 128, 1024), (1, 128, 1025)])
def test_columns_over_a_cluster(shape, dtype, dev):
    """Columns that do not divide among the CTAs (of 520 over eight of 80 the last has none), and the lines between the variants."""
    from cuda_mace_b200 import ops

    U = update(13 + sum(shape), shape, dtype, dev)
    check(ops.orthogonalize(U), U)
    ops.check_status()
