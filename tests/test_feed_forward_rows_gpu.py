"""Rows of the feed-forward block that differ in size: each row of y and of the gradient of x against its OWN size, whichever rows share a
block of 64 with it, and the weights' gradients against the sums of their terms.

Bounds, all in float64.  float32 goes as pairs of fp16 values: an operand is off by at most 2^-22 of itself and by 2^-39 of the largest value
of its block of 64 x 64, where the rows of a block have been brought to one size first.  With s a row's power of two (of x; t: of
dL/dy), a block's largest value is therefore at most 2 max|x / s| of the whole matrix, and that loses 2^-38 max|x / s| s of a value of the row.
The like holds for h / s^2, dg / (s t), du / (s t), and for the contributions x s t and dy s^2 of the sums over rows.  The product of two low
parts (2^-22) is left out, 64 k are summed in 12 truncating additions (2^-22 of the magnitudes) and added with rounding (2^-24)."""
import pytest
import torch

from tests.test_feed_forward_gpu import act_of, case

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "the gpu tests need a CUDA device"
    return torch.device("cuda:0")


def power(x):
    """The power of two of each row's largest value, [M, 1], 2^-127 for subnormal ones and no less than 2^-126 of the largest in its block
    of 64 rows; rows of zeros have the block's largest."""
    most = x.abs().amax(1)
    e = torch.where(most > 0, torch.floor(torch.log2(most.clamp_min(1e-300))).clamp_min(-127.0), -1e3)
    blocks = torch.nn.functional.pad(e, (0, -len(e) % 64), value=-1e3).view(-1, 64)
    top = blocks.amax(1, keepdim=True).expand_as(blocks).reshape(-1)[:len(e)]
    e = torch.where(most > 0, torch.maximum(e, top - 126), top.clamp_min(-126.0))
    return torch.exp2(e)[:, None]


def product(A, B, dA, dB, size_A, size_B):
    """A @ B and its bound.  dA, dB: what the operands are off already.  size_A, size_B: of A's and of B's values (in the shape of either, or
    broadcast), what 2^-38 of is lost beside the 2^-22."""
    K = A.shape[1]
    a, b = 2.0 ** -22 * A.abs() + 2.0 ** -38 * size_A + dA, 2.0 ** -22 * B.abs() + 2.0 ** -38 * size_B + dB
    a, b = a.expand_as(A), b.expand_as(B)
    off = a @ B.abs() + A.abs() @ b + a @ b + (13 * 2.0 ** -22 + (K / 64 + 64) * 2.0 ** -24) * (A.abs() @ B.abs())
    return A @ B, off


def reference(x, wg, wu, wd, gy, activation, low=1.0):
    """Values and bounds of a float32 call, row by row.  low: of the 2^-38 that is lost of a block's largest value."""
    s, t = power(x), power(gy)
    of = lambda v, p: low * (v / p).abs().max() * p  # noqa: E731: the block's largest value at a row's own size
    flat = lambda w: low * w.abs().max()  # noqa: E731
    g, eg = product(x, wg, 0.0, 0.0, of(x, s), flat(wg))
    u, eu = product(x, wu, 0.0, 0.0, of(x, s), flat(wu))
    a, da = act_of(g, activation)
    # |act'| <= 1.13, |act''| <= 0.8; SiLU to 16 roundings of its value, GELU's cumulative distribution to 2^-22
    ea = 1.13 * eg + 2.0 ** -20 * a.abs() + (2.0 ** -22 * g.abs() if activation == "gelu" else 0.0)
    eda = 0.8 * eg + 2.0 ** -20 * (da.abs() + g.abs() * 2.0 ** -4) + 2.0 ** -22
    h = a * u
    eh = ea * (u.abs() + eu) + a.abs() * eu + 2.0 ** -22 * h.abs()
    y, ey = product(h, wd, eh, 0.0, of(h, s * s), flat(wd))
    dh, edh = product(gy, wd.t(), 0.0, 0.0, of(gy, t), flat(wd))
    dg, du = dh * u * da, dh * a
    edg = (dh.abs() + edh) * (u.abs() + eu) * (da.abs() + eda) - dg.abs() + 2.0 ** -22 * dg.abs()
    edu = (dh.abs() + edh) * (a.abs() + ea) - du.abs() + 2.0 ** -22 * du.abs()
    x1, e1 = product(dg, wg.t(), edg, 0.0, of(dg, s * t), flat(wg))
    x2, e2 = product(du, wu.t(), edu, 0.0, of(du, s * t), flat(wu))
    out = {"y": (y, ey), "x": (x1 + x2, e1 + e2 + 2.0 ** -23 * (x1.abs() + x2.abs()))}
    # sums over rows, of rows at the size of their contributions: x s t by dg / (s t), dy s^2 by h / s^2
    for name, A, p, B, eB in (("w_gate", x, s * t, dg, edg), ("w_up", x, s * t, du, edu), ("w_down", gy, s * s, h, eh)):
        v, e = product((A * p).t(), B / p, 0.0, eB / p, low * (A * p).abs().max(), low * (B / p).abs().max())
        out[name] = (v.t(), e.t()) if name == "w_down" else (v, e)
    return {k: (v, e + 2.0 ** -24 * v.abs()) for k, (v, e) in out.items()}


def run(args, activation="silu"):
    from cuda_mace_b200 import ops

    leaves = [t.detach().requires_grad_(True) for t in args[:4]]   # at the addresses that they have
    y = ops.gated_feed_forward(*leaves, activation=activation)
    grads = torch.autograd.grad(y, leaves, args[4])
    ops.check_status()
    return dict(zip(("y", "x", "w_gate", "w_up", "w_down"), [y.detach(), *grads]))


def inside(got, want, names=("y", "x", "w_gate", "w_up", "w_down")):
    for name in names:
        v, bound = want[name]
        assert torch.isfinite(got[name]).all(), name
        off = (got[name].double() - v).abs()
        assert (off <= bound + 1e-37).all(), f"{name}: {(off / bound.clamp_min(1e-300)).max().item():.2f} times the bound"


def of_rows(got, want):
    """The error of each row against its own size, both as norms."""
    return (got.double() - want).norm(dim=1) / want.norm(dim=1).clamp_min(1e-300)


# A row's error as a norm, against its own: ten times the 4e-7 that three products one after the other are off by where all rows have one size.
# The gradient of x has act'(g), off by up to |act''| <= 0.8 of what g is off by, which is in proportion to g: where a row's g are larger than 1, so
# much more, against an act' of 1 (for float32 sums of any kind).
ROW = 2.0 ** -18


def row_bound(name, x, wg):
    g = (x.double() @ wg.double()).abs().amax(1)
    return ROW * (g.clamp_min(1.0) if name == "x" else torch.ones_like(g))


SIZES = [(300, 128, 512), (257, 130, 66), (200, 264, 200), (65, 192, 136), (3000, 136, 520)]


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("M,C,H", SIZES)
def test_rows_spread(M, C, H, activation, dev):
    """Rows of x whose sizes are spread as e^(3 n), n normal, and rows of the gradient of y as e^(2 n)."""
    args = case(M + C + H + 5, M, C, H, F32, dev, spread=3.0)
    n = torch.randn(M, 1, generator=torch.Generator().manual_seed(M), dtype=torch.float64).to(dev)
    args[4] = (args[4].double() * torch.exp(2 * n)).float()
    got, want = run(args, activation), reference(*(v.double() for v in args), activation)
    inside(got, want)
    if activation == "silu":
        for name in ("y", "x"):
            assert (of_rows(got[name], want[name][0]) < row_bound(name, *args[:2])).all(), name


@pytest.mark.parametrize("size", [1e-2, 1e-3, 1e-4, 1e-5, 1e-6, 1e-8, 1e-12])
@pytest.mark.parametrize("M,C,H", [(300, 128, 512), (130, 257, 130)])
def test_single_small_rows(M, C, H, size, dev):
    """One row in 64 that is smaller, in x, in the gradient of y, and in both."""
    args = case(M + 17, M, C, H, F32, dev)
    args[0][5], args[4][5] = args[0][5] * size, args[4][5] * size
    args[0][70] *= size
    args[4][100] *= size
    got, want = run(args), reference(*(v.double() for v in args), "silu")
    inside(got, want)
    for name in ("y", "x"):
        assert (of_rows(got[name], want[name][0]) < row_bound(name, *args[:2])).all(), name


@pytest.mark.parametrize("M", [90, 700])
def test_a_row_is_what_it_is_alone(M, dev):
    """The same rows among others of their size and among ones that are 1e5 times as large: a rounding or two apart."""
    from cuda_mace_b200 import ops

    x, wg, wu, wd, _ = case(23, M, 160, 320, F32, dev)
    want = ops.gated_feed_forward(x * 1e-5, wg, wu, wd)
    mixed = x.clone()
    mixed[1::2] *= 1e-5
    got = ops.gated_feed_forward(mixed, wg, wu, wd)
    assert (of_rows(got[1::2], want[1::2].double()) < ROW).all()


@pytest.mark.parametrize("top", [1e-30, 1e-15, 1.0, 1e12])
def test_rows_far_from_one(top, dev):
    """The largest rows far from one, weights that bring the products back, rows of zeros and subnormal rows among them."""
    M, C, H = 200, 136, 200
    x, wg, wu, wd, gy = case(29, M, C, H, F32, dev, spread=2.0)
    x[3], gy[9], x[64:128] = 0, 0, 0
    x = x * top
    x[130] = torch.linspace(-1e-40, 1e-40, C, device=dev)
    args = [x, wg / top, wu / top, wd, gy]
    got = run(args)
    want = reference(*(v.double() for v in args), "silu")
    assert not got["y"][3].any() and not got["y"][64:128].any() and not got["x"][9].any()
    inside(got, want)


@pytest.mark.parametrize("size", [1e4, 1e8])
def test_rows_without_a_gradient(size, dev):
    """Rows that do not count (a gradient of zeros, as of padding) and are far larger than those that do; rows of zeros with a large gradient."""
    args = case(37, 192, 136, 200, F32, dev)
    for rows in (slice(3, 20), slice(64, 70)):
        args[0][rows] *= size
        args[4][rows] = 0
    args[0][130:140] = 0
    args[4][130:140] *= size
    got = run(args)
    few = [args[0].clone(), *args[1:4], args[4].clone()]
    for k in (0, 4):
        few[k][3:20], few[k][64:70], few[k][130:140] = 0, 0, 0
    inside(got, reference(*(v.double() for v in args), "silu"))
    inside(got, reference(*(v.double() for v in few), "silu"), ("w_gate", "w_up", "w_down"))


@pytest.mark.parametrize("M,C,H", [(1, 300, 17), (9, 130, 56), (3, 352, 170)])
def test_rows_as_pairs_bfloat16(M, C, H, dev):
    """bfloat16 operands that go as pairs keep what bfloat16's own exponent keeps: results are off by their rounding."""
    from cuda_mace_b200 import ops

    args = case(M + 31, M, C, H, BF16, dev, spread=6.0)
    leaves = [t.clone().requires_grad_(True) for t in args[:4]]
    y = ops.gated_feed_forward(*leaves)
    gx = torch.autograd.grad(y, leaves[0], args[4])[0]
    want = reference(*(v.double() for v in args), "silu")
    for got, name in ((y.detach(), "y"), (gx, "x")):
        v, bound = want[name]
        assert ((got.double() - v).abs() <= bound + 2.0 ** -8 * (v.abs() + bound) + 1e-37).all(), name


@pytest.mark.parametrize("M,C,H", [(100, 256, 2048), (64, 264, 1500)])
def test_rows_of_split_sums(M, C, H, dev):
    """Sums over the hidden columns that are split over the SMs."""
    args = case(M + 41, M, C, H, F32, dev, spread=4.0)
    got, want = run(args), reference(*(v.double() for v in args), "silu")
    inside(got, want)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("M,C,H", [(129, 132, 68), (129, 133, 70)])
def test_layouts_of_spread_rows(M, C, H, apart, dev):
    """Widths and addresses that vector loads cannot take, and each gradient alone."""
    from cuda_mace_b200 import ops

    args = case(M + 51, M, C, H, F32, dev, spread=3.0)
    if apart:
        for i, v in enumerate(args):
            room = torch.zeros(v.numel() + 1, device=dev)
            room[1:] = v.flatten()
            args[i] = room[1:].view(v.shape)
    want = reference(*(v.double() for v in args), "silu")
    got = run(args)
    inside(got, want)
    for k, name in enumerate(("x", "w_gate", "w_up", "w_down")):
        leaves = [v.detach().requires_grad_(k == i) for i, v in enumerate(args[:4])]
        (g,) = torch.autograd.grad(ops.gated_feed_forward(*leaves), leaves[k], args[4])
        assert torch.equal(g, got[name]), name
        inside({name: g}, want, (name,))


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("M,C,H", [(130, 128, 200), (150, 200, 136)])
@pytest.mark.parametrize("size", [1e15, 1e20, 1e30, 3e37])
def test_rows_whose_hidden_values_overflow(M, C, H, size, activation, dev):
    """Rows so large that their own h, or y, is no float32 value, beside rows that are not: those keep theirs."""
    args = case(M + 83, M, C, H, F32, dev)
    large = torch.zeros(M, dtype=torch.bool, device=dev)
    large[[2, 40, 70, M - 1]] = True
    few = [t.clone() for t in args]
    few[0][large], few[4][large] = 0, 0
    args[0][large] = (args[0][large].double() * size / 8).clamp(-3e38, 3e38).float()
    want = reference(*(v.double() for v in few), activation)   # of the other rows
    got = run(args, activation)
    for name in ("y", "x"):
        v, bound = want[name]
        off = (got[name].double() - v).abs()[~large]
        assert torch.isfinite(off).all() and (off <= bound[~large] + 1e-37).all(), name
    # rows that do not count leave the weights' gradients alone, as far as zero times their h is one
    if size < 1e18:
        args[4][large] = 0
        inside(run(args, activation), want, ("w_gate", "w_up", "w_down"))


@pytest.mark.parametrize("M,C,H", [(130, 128, 200), (150, 200, 136)])
def test_weights_and_rows_far_apart(M, C, H, dev):
    """Weights of 1e20: half of the rows are small enough for them, the others overflow."""
    x, wg, wu, wd, gy = case(M + 89, M, C, H, F32, dev)
    wg, wu = wg * 1e20, wu * 1e20
    x[::2] *= 1e-20
    few = [x.clone(), wg, wu, wd, gy.clone()]
    few[0][1::2], few[4][1::2] = 0, 0
    want = reference(*(v.double() for v in few), "silu")
    got = run([x, wg, wu, wd, gy])
    for name in ("y", "x"):
        v, bound = want[name]
        off = (got[name].double() - v).abs()[::2]
        assert torch.isfinite(off).all() and (off <= bound[::2] + 1e-37).all(), name


def test_contributions_of_large_rows(dev):
    """Rows of 1e20 with gradients of 1e-25 and weights that keep h a float32 value: the weights' gradients are finite sums of all rows."""
    M, C, H = 200, 128, 136
    x, wg, wu, wd, gy = case(97, M, C, H, F32, dev)
    wg, wu = wg * 1e-12, wu * 1e-12
    x[::3] *= 1e20
    gy[::3] *= 1e-25
    args = [x, wg, wu, wd, gy]
    inside(run(args), reference(*(v.double() for v in args), "silu"))
