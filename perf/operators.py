"""The operators that train and serve a model's dense blocks, as cases that can be timed.

Kinds of cases (`kind`) and what one pass is:

* ``feed_forward``: the gated feed-forward block on rows of node features,
  ``y = (act(x w_gate) * (x w_up)) w_down`` with x [rows, width], w_gate and w_up [width, hidden], w_down [hidden, width]:
    - ``how`` = ``forward``: the block alone, as an evaluation asks for it;
    - ``how`` = ``train``: the block, then the gradients of x and of the three weights for a given gradient of y.
* ``orthogonalize``: the update of a stack of weight matrices [count, rows, columns], brought near its orthogonal factor by five
  Newton-Schulz products: ``X_0 = U / (|U| + eps)``, ``X <- a X + (b A + c A A) X`` with ``A = X X^T``, which is how the weights of the
  block, of Linear and of ElementalLinear are stepped by an optimiser that wants every direction of an update to count alike.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7


def listed():
    def ff(name, rows, width, hidden, dtype, how, activation="silu"):
        return dict(name=name, kind="feed_forward", rows=rows, width=width, hidden=hidden, dtype=dtype, how=how,
                    activation=activation)

    def ortho(name, count, rows, columns, dtype):
        return dict(name=name, kind="orthogonalize", count=count, rows=rows, columns=columns, dtype=dtype)

    return [
        # one row, a block whose weights are all there is to read: the service of single requests
        ff("ff 1 row bf16", 1, 1024, 4096, "bf16", "forward"),
        # a small molecule-sized cell, the width and the hidden width of a 128-channel model's readout
        ff("ff 192 f32", 192, 128, 512, "f32", "forward"),
        # a box of water, ragged sizes, the other activation
        ff("ff 2999 odd bf16 gelu", 2999, 250, 1001, "bf16", "forward", "gelu"),
        # the most atoms of one card in the precision the models run in
        ff("ff 64000 f32", 64000, 128, 512, "f32", "forward"),
        # a training batch of structures, float32
        ff("ff train 15999 f32", 15999, 128, 512, "f32", "train"),
        # the widest block, bf16, forward and training
        ff("ff 16384 bf16", 16384, 1024, 4096, "bf16", "forward"),
        ff("ff train 8192 bf16", 8192, 1024, 4096, "bf16", "train"),
        # the smallest stack: the radial perceptron's hidden matrices of two layers
        ortho("ortho 4x64x64 f32", 4, 64, 64, "f32"),
        # an ElementalLinear's matrices: 10 elements, 4 degrees, 128 channels
        ortho("ortho 40x128x128 f32", 40, 128, 128, "f32"),
        # the block's projections at a 128-channel model's widths
        ortho("ortho 3x128x512 bf16", 3, 128, 512, "bf16"),
        # odd sides, more rows than columns
        ortho("ortho 1x1001x250 f32", 1, 1001, 250, "f32"),
        # the projections of the widest block
        ortho("ortho 2x1024x4096 bf16", 2, 1024, 4096, "bf16"),
    ]


def _size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    if c["kind"] == "feed_forward":
        return (18 if c["how"] == "train" else 6) * c["rows"] * c["width"] * c["hidden"]
    small, large = sorted((c["rows"], c["columns"]))
    return STEPS * c["count"] * (3 * small * small * large + small ** 3)


def draw(rng):
    kind = rng.choice(["feed_forward", "feed_forward", "orthogonalize"])
    dtype = rng.choice(["f32", "bf16"])
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        if kind == "feed_forward":
            c = dict(kind=kind, rows=_size(rng, 1, 64000), width=_size(rng, 16, 1024), hidden=_size(rng, 16, 4096), dtype=dtype,
                     how=rng.choice(["forward", "train"]), activation=rng.choice(["silu", "gelu"]))
            # half of the blocks have the widths that models are built with
            if rng.random() < 0.5:
                c["width"] = max(32, c["width"] // 32 * 32)
                c["hidden"] = rng.choice([2, 4]) * c["width"]
        else:
            c = dict(kind=kind, count=_size(rng, 1, 64), rows=_size(rng, 16, 2048), columns=_size(rng, 16, 4096), dtype=dtype)
            if rng.random() < 0.5:
                c["rows"], c["columns"] = max(32, c["rows"] // 32 * 32), max(32, c["columns"] // 32 * 32)
        if _cost(c) <= most:
            return c


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "feed_forward":
        m, c, h = case["rows"], case["width"], case["hidden"]
        train = case["how"] == "train"
        # features of unit size whose channels differ in scale, as contractions of messages leave them
        x = _normal(gen, m, c) * torch.exp(0.3 * _normal(gen, c))
        s = dict(case, x=x.to(dt), w_gate=(_normal(gen, c, h) / math.sqrt(c)).to(dt), w_up=(_normal(gen, c, h) / math.sqrt(c)).to(dt),
                 w_down=(_normal(gen, h, c) / math.sqrt(h)).to(dt))
        if train:
            s["gy"] = _normal(gen, m, c).to(dt)
            for k in ("x", "w_gate", "w_up", "w_down"):
                s[k].requires_grad_(True)
        return s
    n, r, c = case["count"], case["rows"], case["columns"]
    # a gradient of a product: features^T times gradients of its result, over rows of a batch; features differ in scale
    t = min(4096, 2 * max(r, c))
    a = _normal(gen, n, t, r) * torch.exp(0.5 * _normal(gen, n, 1, r))
    b = _normal(gen, n, t, c) * torch.exp(0.5 * _normal(gen, n, 1, c))
    return dict(case, update=(a.transpose(1, 2) @ b / t).to(dt))


def _gate(g, activation):
    """act(g) and its derivative."""
    if activation == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_feed_forward(s):
    dt = s["x"].dtype
    x, wg, wu, wd = (s[k].detach().float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg, x @ wu
    a, da = _gate(g, s["activation"])
    h = a * u
    y = (h @ wd).to(dt)
    if s["how"] == "forward":
        return {"y": y}
    gy = s["gy"].float()
    gh = gy @ wd.t()
    gg, gu = gh * u * da, gh * a
    return {"y": y, "grad_x": (gg @ wg.t() + gu @ wu.t()).to(dt), "grad_gate": (x.t() @ gg).to(dt), "grad_up": (x.t() @ gu).to(dt),
            "grad_down": (h.t() @ gy).to(dt)}


def _plain_orthogonalize(s):
    a, b, c = COEFFICIENTS
    u = s["update"].float()
    tall = u.shape[1] > u.shape[2]
    x = u.transpose(1, 2) if tall else u
    x = x / (torch.sqrt((x * x).sum(dim=(1, 2), keepdim=True)) + EPS)
    for _ in range(STEPS):
        gram = x @ x.transpose(1, 2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return {"out": (x.transpose(1, 2) if tall else x).to(s["update"].dtype).contiguous()}


def run(state):
    if not own:
        with torch.no_grad():
            return _plain_feed_forward(state) if state["kind"] == "feed_forward" else _plain_orthogonalize(state)
    from cuda_mace_b200 import ops

    if state["kind"] == "orthogonalize":
        return {"out": ops.orthogonalize(state["update"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)}
    leaves = tuple(state[k] for k in ("x", "w_gate", "w_up", "w_down"))
    y = ops.gated_feed_forward(*leaves, activation=state["activation"])
    if state["how"] == "forward":
        return {"y": y}
    gx, gg, gu, gd = torch.autograd.grad(y, leaves, state["gy"])
    return {"y": y, "grad_x": gx, "grad_gate": gg, "grad_up": gu, "grad_down": gd}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "feed_forward":
        m, c, h = case["rows"], case["width"], case["hidden"]
        rows, weights = m * c, 3 * c * h
        if case["how"] == "forward":
            return {"bytes": size * (2 * rows + weights), "flops": 6 * m * c * h}
        # x, the gradient of y and the weights in; y, the gradient of x and the weights' gradients out
        return {"bytes": size * (4 * rows + 2 * weights), "flops": 18 * m * c * h}
    # per step a symmetric product X X^T and a symmetric square (half of each needs forming), and one full product
    return {"bytes": 2 * size * case["count"] * case["rows"] * case["columns"], "flops": _cost(case)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "feed_forward":
        leaves = [s[k].detach().double().requires_grad_(True) for k in ("x", "w_gate", "w_up", "w_down")]
        x, wg, wu, wd = leaves
        act = torch.nn.functional.silu if case["activation"] == "silu" else torch.nn.functional.gelu
        y = torch.einsum("mh,hc->mc", act(torch.einsum("mc,ch->mh", x, wg)) * torch.einsum("mc,ch->mh", x, wu), wd)
        if case["how"] == "forward":
            return {"y": y.detach()}
        gx, gg, gu, gd = torch.autograd.grad(y, leaves, s["gy"].double())
        return {"y": y.detach(), "grad_x": gx, "grad_gate": gg, "grad_up": gu, "grad_down": gd}
    # the same polynomial of the singular values, X <- X (a + b X^T X + c (X^T X)^2), from the right where that is smaller
    a, b, c = COEFFICIENTS
    x = s["update"].double()
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + EPS)
    one = torch.eye(min(x.shape[1:]), dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        if x.shape[1] <= x.shape[2]:
            w = torch.einsum("nik,njk->nij", x, x)
            x = torch.einsum("nij,njk->nik", a * one + torch.einsum("nij,njk->nik", w, b * one + c * w), x)
        else:
            w = torch.einsum("nki,nkj->nij", x, x)
            x = torch.einsum("nij,njk->nik", x, a * one + torch.einsum("nij,njk->nik", w, b * one + c * w))
    return {"out": x}
