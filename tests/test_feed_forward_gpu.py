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


def run_all(x, wg, wu, wd, gy, activation="silu"):
    from cuda_mace_b200 import ops

    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = ops.gated_feed_forward(*leaves, activation=activation)
    return [y.detach()] + list(torch.autograd.grad(y, leaves, gy))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [1, 3, 4, 5, 8, 9])
@pytest.mark.parametrize("C,H", [(32, 64), (33, 70), (1030, 36), (36, 1030), (1, 8)])
def test_few_rows(M, C, H, dtype, dev):
    """Both sides of the line between the pass over the weights and the tiles, more of W's rows than are kept at once."""
    from cuda_mace_b200 import ops

    x, wg, wu, wd, _ = case(M + C + H + 7, M, C, H, dtype, dev)
    y = ops.gated_feed_forward(x, wg, wu, wd)
    inside(y, reference(*(t.double() for t in (x, wg, wu, wd)), None, "silu", dtype)["y"])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [6, 70])
def test_layouts(M, dtype, dev):
    """Leading dimensions, strides, addresses off a boundary: the values of a call on contiguous copies."""
    from cuda_mace_b200 import ops

    C, H = 64, 96
    x, wg, wu, wd, gy = case(M, M, C, H, dtype, dev)
    want = run_all(x, wg, wu, wd, gy)
    as_rows = ops.gated_feed_forward(x.view(2, M // 2, C), wg, wu, wd)
    assert as_rows.shape == (2, M // 2, C) and torch.equal(as_rows.view(M, C), want[0])
    flipped = [x.t().contiguous().t(), wg.t().contiguous().t(), wu.t().contiguous().t(), wd.t().contiguous().t(), gy.t().contiguous().t()]
    for a, b in zip(run_all(*flipped), want):
        assert torch.equal(a, b)
    off = []
    for t in (x, wg, wu, wd, gy):
        room = torch.zeros(t.numel() + 1, dtype=dtype, device=dev)
        room[1:].copy_(t.reshape(-1))
        off.append(room[1:].view(t.shape))   # 2 or 4 bytes off a boundary of 16
    leaves = [t.requires_grad_(True) for t in off[:4]]
    y = ops.gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, off[4])
    want_ref = reference(*(t.double() for t in (x, wg, wu, wd, gy)), "silu", dtype)
    inside(y.detach(), want_ref["y"])
    for name, g in zip(("x", "w_gate", "w_up", "w_down"), grads):
        inside(g, want_ref[name])
    # one row that all positions of an expanded x share, and the gradient of a sum (an expanded one)
    one = x[:1].clone().requires_grad_(True)
    y = ops.gated_feed_forward(one.expand(M, C), wg, wu, wd)
    (g,) = torch.autograd.grad(y.float().sum(), one)
    assert g.shape == (1, C) and torch.isfinite(g).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_no_rows(dtype, dev):
    x, wg, wu, wd, gy = case(3, 1, 24, 40, dtype, dev)
    y, gx, gg, gu, gd = run_all(x[:0], wg, wu, wd, gy[:0])
    assert y.shape == (0, 24) and gx.shape == (0, 24)
    for g, w in ((gg, wg), (gu, wu), (gd, wd)):
        assert g.shape == w.shape and not g.any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,C,H", [(40, 32, 48), (3000, 130, 200)])
def test_gradients_of_some(M, C, H, dtype, dev):
    """Each gradient alone has the bits that it has among all."""
    from cuda_mace_b200 import ops

    t = case(11, M, C, H, dtype, dev)
    want = run_all(*t)
    for which in range(4):
        leaves = [v.clone().requires_grad_(k == which) for k, v in enumerate(t[:4])]
        (g,) = torch.autograd.grad(ops.gated_feed_forward(*leaves), leaves[which], t[4])
        assert torch.equal(g, want[1 + which]), which
    # one matrix as both projections: its gradient is the sum of theirs
    w = t[1].clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.gated_feed_forward(t[0], w, w, t[3]), w, t[4])
    both = run_all(t[0], t[1], t[1], t[3], t[4])
    assert torch.equal(g, both[2] + both[3])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [5, 200])
def test_rows_that_are_not_finite(M, dtype, dev):
    """An infinity or a NaN in a row spoils that row alone, whichever block of rows shares a scale with it."""
    C, H = 48, 80
    x, wg, wu, wd, gy = case(21, M, C, H, dtype, dev)
    want = run_all(x, wg, wu, wd, gy)
    bad = x.clone()
    bad[1, 3], bad[3, 0], bad[4, 47] = float("inf"), float("nan"), -float("inf")
    got = run_all(bad, wg, wu, wd, gy)
    spoiled = torch.tensor([1, 3, 4], device=dev)
    fine = torch.ones(M, dtype=torch.bool, device=dev)
    fine[spoiled] = False
    for a, b in ((got[0], want[0]), (got[1], want[1])):
        assert not torch.isfinite(a[spoiled]).all(dim=1).any()
        scale = b[fine].abs().max()
        # other finite values of the block set its scale as before: but for the spoiled values' own, which may have been the largest
        assert torch.isfinite(a[fine]).all() and (a[fine] - b[fine]).abs().max() <= 2.0 ** -20 * scale
    for g in got[2:]:
        assert not torch.isfinite(g).all()


@pytest.mark.parametrize("M", [300, 5])
def test_ranges_float32(M, dev):
    """Blocks far from each other in size, and far from one: a block's scale is its own."""
    C, H = 192, 130
    x, wg, wu, wd, gy = case(31, M, C, H, F32, dev)
    x[:64] *= 1e-20
    x[64:128] *= 1e6
    x[:, 64:128] *= 1e-6
    for k, t in ((1e-12, 1e3), (1e6, 1e-9)):
        args = [x * k, wg * t, wu, wd * 10, gy]
        want = reference(*(v.double() for v in args), "silu", F32)
        got = run_all(*args)
        for name, g in zip(("y", "x", "w_gate", "w_up", "w_down"), got):
            v, bound = want[name]
            # below the normal range nothing is held; what is summed is of one row's or column's size
            assert (g.double() - v).abs().le(bound + 1e-30).all(), name
        if M > 128:   # rows of a block of their own: as if they were alone
            from cuda_mace_b200 import ops

            assert torch.equal(got[0][:64], ops.gated_feed_forward(args[0][:64], *args[1:4]))


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_against_differences(activation, dev):
    """The gradient along a direction is the central difference of the operator's own values: third derivatives are O(1) here, so the
    quotient is off by O(h^2) of the sum of magnitudes and by the rounding of both values over 2 h."""
    from cuda_mace_b200 import ops

    M, C, H, h = 50, 40, 72, 2.0 ** -6
    t = case(41, M, C, H, F32, dev)
    d = case(42, M, C, H, F32, dev)
    got = run_all(*t, activation=activation)
    for which in range(4):
        def at(s):
            args = [v + s * h * d[k] if k == which else v for k, v in enumerate(t[:4])]
            return (ops.gated_feed_forward(*args, activation=activation).double() * t[4].double()).sum()
        quotient = (at(1.0) - at(-1.0)) / (2 * h)
        slope = (got[1 + which].double() * d[which].double()).sum()
        size = (got[1 + which].abs().double() * d[which].abs().double()).sum()
        noise = (got[0].abs().double() * t[4].abs().double()).sum() * 2.0 ** -18 / h
        assert (quotient - slope).abs() <= 10 * h * h * size + noise, which


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,C,H", [(4, 64, 64), (100, 100, 60), (4000, 64, 128)])
def test_same_bits(M, C, H, dtype, dev):
    t = case(51, M, C, H, dtype, dev)
    first = run_all(*t)
    for _ in range(3):
        for a, b in zip(run_all(*t), first):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [4, 700])
def test_streams(M, dtype, dev):
    """Two calls at once on streams of their own, and a call on another stream than the inputs'."""
    from cuda_mace_b200 import ops

    sets = [case(60 + k, M, 96, 160, dtype, dev) for k in range(2)]
    want = [run_all(*t) for t in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(4):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k] = run_all(*sets[k])
        torch.cuda.synchronize()
        for k in range(2):
            for a, b in zip(got[k], want[k]):
                assert torch.equal(a, b)
    x = sets[0][0] * 1.0   # on the default stream, not waited for on the host
    streams[0].wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(streams[0]):
        y = ops.gated_feed_forward(x, *sets[0][1:4])
    torch.cuda.current_stream().wait_stream(streams[0])
    assert torch.equal(y, want[0][0])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M", [3, 500])
def test_recorded(M, dtype, dev):
    """Forward and backward recorded as graphs and replayed on new values; two graphs of the same pool."""
    from cuda_mace_b200 import ops

    sets = [case(70 + k, M, 64, 136, dtype, dev) for k in range(3)]
    want = [run_all(*t) for t in sets]
    static = [t.clone().requires_grad_(k < 4) for k, t in enumerate(sets[0])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.gated_feed_forward(*static[:4])
        torch.autograd.grad(y, static[:4], static[4])
    torch.cuda.current_stream().wait_stream(side)
    eager = ops.gated_feed_forward(*static[:4])   # an eager graph of the same leaves lives on
    graphs, results = [], []
    pool = None
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            y = ops.gated_feed_forward(*static[:4])
            results.append([y.detach()] + list(torch.autograd.grad(y, static[:4], static[4])))
        pool = g.pool()
        graphs.append(g)
    for k in (1, 2, 0):
        with torch.no_grad():
            for a, b in zip(static, sets[k]):
                a.copy_(b)
        for g, r in zip(graphs, results):
            g.replay()
            for a, b in zip(r, want[k]):
                assert torch.equal(a, b)
    assert torch.equal(eager.detach(), want[0][0])


def test_differentiable_once(dev):
    from cuda_mace_b200 import ops

    t = [v.requires_grad_(True) for v in case(81, 20, 16, 24, F32, dev)[:4]]
    y = ops.gated_feed_forward(*t)
    (g,) = torch.autograd.grad(y.sum(), t[0], create_graph=True)
    with pytest.raises(RuntimeError):   # torch's own words: no path leads there
        torch.autograd.grad(g.sum(), t[1], retain_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


def test_module(dev):
    from cuda_mace_b200 import ops

    x, wg, wu, wd, gy = case(91, 30, 32, 64, F32, dev)
    block = ops.GatedFeedForward(wg, wu, wd, activation="gelu")
    assert {n for n, _ in block.named_parameters()} == {"w_gate", "w_up", "w_down"}
    y = block(x)
    assert torch.equal(y.detach(), run_all(x, wg, wu, wd, gy, "gelu")[0])
    y.backward(gy)
    assert torch.equal(block.w_down.grad, run_all(x, wg, wu, wd, gy, "gelu")[4])


def test_refusals_on_the_device(dev):
    from cuda_mace_b200 import _abi, ops

    x, wg, wu, wd, _ = case(95, 4, 16, 24, F32, dev)
    with pytest.raises(TypeError, match="one type"):
        ops.gated_feed_forward(x, wg.bfloat16(), wu, wd)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ops.gated_feed_forward(*(t.double() for t in (x, wg, wu, wd)))
    with pytest.raises(RuntimeError, match="shape mismatch"):
        ops.gated_feed_forward(x, wg, wu[:, :-1], wd)
    with pytest.raises(RuntimeError, match="shape mismatch"):
        ops.gated_feed_forward(x[:, :-1], wg, wu, wd)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.gated_feed_forward(x, wg.cpu(), wu, wd)
    y = torch.full_like(x, 7.0)
    ws = torch.empty(1 << 16, dtype=torch.uint8, device=dev)
    args = (x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), 4, 16, 24, 0, y.data_ptr())
    for tail, what in (((0, 1 << 16, 0, 0), "null pointer"), ((ws.data_ptr() + 16, 1 << 15, 0, 0), "aligned"), ((ws.data_ptr(), 16, 0, 0), "needed")):
        with pytest.raises(RuntimeError, match=what):
            _abi.call("cmace_gated_ff_fwd_f32", *args, *tail)
    torch.cuda.synchronize()
    assert (y == 7.0).all()


def test_block_trained_with_orthogonalised_updates(dev):
    """The dense operators together, as an optimiser step uses them: block, gradients, orthogonalised updates of the three matrices."""
    from cuda_mace_b200 import ops

    x, wg, wu, wd, gy = case(99, 400, 64, 128, F32, dev)
    block = ops.GatedFeedForward(wg, wu, wd)
    momentum = {n: torch.zeros_like(p) for n, p in block.named_parameters()}
    want = {n: p.detach().double().clone() for n, p in block.named_parameters()}
    want_m = {n: torch.zeros_like(p) for n, p in want.items()}
    for step in range(3):
        block.zero_grad()
        block(x).backward(gy)
        ref = reference(x.double(), want["w_gate"], want["w_up"], want["w_down"], gy.double(), "silu", F32)
        with torch.no_grad():
            for n, p in block.named_parameters():
                momentum[n].mul_(0.9).add_(p.grad)
                p.sub_(0.02 * ops.orthogonalize(momentum[n]))
        for n in want:
            want_m[n] = 0.9 * want_m[n] + ref[n][0]
            u = want_m[n] / (want_m[n].norm() + 1e-7)
            for _ in range(5):
                s = u @ u.t()
                u = 3.4445 * u + (-4.7750 * s + 2.0315 * s @ s) @ u
            want[n] = want[n] - 0.02 * u
    ops.check_status()
    for n, p in block.named_parameters():
        # a step moves a weight by at most 0.02 * 1.3 a singular direction; the gradients' 1e-6 are enlarged by up to 485 in the smallest
        assert rel_err(p, want[n]) < 1e-4, n


def test_forward_mode_is_refused(dev):
    from torch.autograd import forward_ad

    from cuda_mace_b200 import ops

    t = list(case(82, 20, 16, 24, F32, dev)[:4])
    with forward_ad.dual_level():
        for i in range(4):
            dual = list(t)
            dual[i] = forward_ad.make_dual(t[i], torch.ones_like(t[i]))
            with pytest.raises(NotImplementedError):
                ops.gated_feed_forward(*dual)
        ops.gated_feed_forward(*t)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,C,H", [(9, 16, 16), (16, 32, 512), (17, 40, 200), (100, 128, 512), (33, 100, 301), (40, 127, 65), (1, 20, 900), (7, 64, 64),
                                   (700, 128, 128), (300, 8, 8), (64, 36, 1030), (3000, 33, 70), (2500, 32, 64), (400, 96, 1100), (50, 4, 2), (20, 24, 20000), (3, 16, 5000)])
def test_some_rows(M, C, H, dtype, apart, dev):
    """Sizes on both sides of where one kernel has the whole block; `apart`: operands one element behind an aligned address."""
    from cuda_mace_b200 import ops

    t = case(M + C + H + 1, M, C, H, dtype, dev)[:4]
    if apart:
        for i, v in enumerate(t):
            buffer = torch.full((v.numel() + 1,), float("nan"), dtype=dtype, device=dev)
            buffer[1:] = v.flatten()
            t[i] = buffer[1:].view(v.shape)
    y = ops.gated_feed_forward(*t)
    inside(y, reference(*(v.double() for v in t), None, "silu", dtype)["y"])
    assert torch.equal(y, ops.gated_feed_forward(*t))
    # what lies behind the last row is not written: the C entry with room behind y
    from cuda_mace_b200 import _abi

    f32 = dtype == F32
    room = torch.full((M * C + 64,), 7.0, dtype=dtype, device=dev)
    n = _abi.call("cmace_gated_ff_workspace_bytes", int(f32), M, C, H, 0)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device=dev)   # NaN wherever a value that was never written is read
    stream = torch.cuda.current_stream().cuda_stream
    _abi.call("cmace_gated_ff_fwd_" + ("f32" if f32 else "bf16"), *(v.data_ptr() for v in t), M, C, H, 0, room.data_ptr(), ws.data_ptr(), n, 0, stream)
    assert torch.equal(room[:M * C].view(M, C), y) and (room[M * C:] == 7.0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,C,H", [(40, 32, 64), (40, 120, 500)])
def test_some_rows_that_are_not_finite(M, C, H, dtype, dev):
    from cuda_mace_b200 import ops

    t = case(93, M, C, H, dtype, dev)[:4]
    want = ops.gated_feed_forward(*t)
    x = t[0].clone()
    x[0, 3], x[17, C - 1], x[39, 0] = float("nan"), float("inf"), float("-inf")
    got = ops.gated_feed_forward(x, *t[1:])
    bad = torch.zeros(M, dtype=torch.bool, device=dev)
    bad[[0, 17, 39]] = True
    assert torch.equal(got[~bad], want[~bad])
    assert not torch.isfinite(got[bad]).all(1).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,C,H", [(100, 256, 2048), (64, 264, 1500), (9, 130, 4100), (300, 33, 3001), (700, 132, 1024)])
def test_sums_over_many_hidden_columns(M, C, H, dtype, dev):
    """Few rows and long sums, which are split, for y and the gradient of x."""
    t = case(M + C + H + 2, M, C, H, dtype, dev)
    got, again = run_all(*t, "silu"), run_all(*t, "silu")
    want = reference(*(v.double() for v in t), "silu", dtype)
    for name, a, b in zip(("y", "x", "w_gate", "w_up", "w_down"), got, again):
        inside(a, want[name])
        assert torch.equal(a, b)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("M,C,H", [(1, 64, 128), (1, 300, 17), (9, 130, 56), (3, 352, 170), (16, 200, 32), (8, 33, 63), (2, 1024, 256), (9, 36, 2931), (1, 1000, 1500)])
def test_few_hidden_values_bfloat16(M, C, H, activation, dev):
    """Few hidden values are not rounded to bfloat16 between the products: every result is off by its own rounding and float32's part."""
    t = case(M + C + H + 3, M, C, H, BF16, dev)
    got = run_all(*t, activation)
    want = reference(*(v.double() for v in t), activation, F32)
    for name, a in zip(("y", "x", "w_gate", "w_up", "w_down"), got):
        v, bound = want[name]
        inside(a, (v, bound + 2.0 ** -8 * (v.abs() + bound)))


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("M,C,H", [(5000, 16, 24), (700, 32, 32)])
def test_gradients_of_few_weights_bfloat16(M, C, H, activation, dev):
    """Neither are they where the weights are few, for the gradients (the forward pass may)."""
    t = case(M + C + H + 4, M, C, H, BF16, dev)
    got = run_all(*t, activation)
    want = reference(*(v.double() for v in t), activation, F32)
    for name, a in zip(("x", "w_gate", "w_up", "w_down"), got[1:]):
        v, bound = want[name]
        inside(a, (v, bound + 2.0 ** -8 * (v.abs() + bound)))
