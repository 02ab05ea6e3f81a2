"""The dense operators under tracers and function transforms: the values of a plain call, or a refusal, never a recording that computes nothing."""
import os
import subprocess
import sys

import pytest
import torch

from tests.test_feed_forward_gpu import case

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16 = torch.float32, torch.bfloat16


def operands(M=20, dtype=F32):
    return case(7, M, 16, 24, dtype, "cuda")


FIRST = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from cuda_mace_b200 import ops

with FakeTensorMode():
    x, w, d = (torch.randn(*s, device="cuda") for s in ((20, 16), (16, 24), (24, 16)))
    y = ops.gated_feed_forward(x, w, w, d)
    assert tuple(y.shape) == (20, 16) and type(y) is not torch.Tensor
x, w, d = (torch.randn(*s, device="cuda") for s in ((20, 16), (16, 24), (24, 16)))
assert torch.isfinite(ops.gated_feed_forward(x, w, w, d)).all()
ops.check_status()
"""


def test_traced_before_the_first_call():
    """What a tracer makes for itself is not kept for the calls that follow."""
    r = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_recorded_graph_computes(dtype):
    from torch.fx.experimental.proxy_tensor import make_fx

    from cuda_mace_b200 import ops

    x, wg, wu, wd, _ = operands(dtype=dtype)
    ops.gated_feed_forward(x, wg, wu, wd)
    graph = make_fx(lambda a, b: ops.gated_feed_forward(a, b, wu, wd, activation="gelu"))(x, wg)
    for k in range(2):
        a, b = x + k, wg * (1 + k)
        assert torch.equal(graph(a, b), ops.gated_feed_forward(a, b, wu, wd, activation="gelu"))


@pytest.mark.parametrize("M", [3, 200])
def test_compiled(M):
    from cuda_mace_b200 import ops

    x, wg, wu, wd, gy = operands(M)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    step = torch.compile(lambda *t: ops.gated_feed_forward(*t) * 2, backend="aot_eager")
    want = ops.gated_feed_forward(*leaves) * 2
    got = step(*leaves)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, gy), torch.autograd.grad(want, leaves, gy)):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(step(*leaves), want)


def test_batched_by_transforms():
    from cuda_mace_b200 import ops

    x, wg, wu, wd, gy = operands()
    xs, ws = torch.stack([x, x * 2, -x]), torch.stack([wg, wu, wg + wu])
    got = torch.func.vmap(lambda a: ops.gated_feed_forward(a, wg, wu, wd))(xs)
    assert torch.equal(got, torch.stack([ops.gated_feed_forward(a, wg, wu, wd) for a in xs]))
    got = torch.func.vmap(lambda w: ops.gated_feed_forward(x, w, wu, wd))(ws)
    assert torch.equal(got, torch.stack([ops.gated_feed_forward(x, w, wu, wd) for w in ws]))
    leaf = x.clone().requires_grad_(True)
    grads = torch.stack([gy, gy * 3])
    (got,) = torch.autograd.grad(ops.gated_feed_forward(leaf, wg, wu, wd), leaf, grads, is_grads_batched=True)
    want = [torch.autograd.grad(ops.gated_feed_forward(leaf, wg, wu, wd), leaf, g)[0] for g in grads]
    assert torch.equal(got, torch.stack(want))


def test_refused():
    from torch.fx.experimental.proxy_tensor import make_fx

    from cuda_mace_b200 import ops

    x, wg, wu, wd, _ = operands()
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: ops.gated_feed_forward(a, wg, wu, wd).sum())(x)
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda a: ops.gated_feed_forward(a, wg, wu, wd), (x,), (x,))
    with pytest.raises(RuntimeError, match="tracer"):
        make_fx(lambda u: ops.orthogonalize(u))(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(ops.orthogonalize)(x[None])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda u: ops.orthogonalize(u).sum())(x)


def test_kept_elsewhere_and_formed_again():
    """Saved tensors on the host, and a checkpointed block."""
    from torch.utils.checkpoint import checkpoint

    from cuda_mace_b200 import ops

    x, wg, wu, wd, gy = operands(90)
    block = ops.GatedFeedForward(wg, wu, wd)
    leaf = x.requires_grad_(True)
    (want,) = torch.autograd.grad(block(leaf), leaf, gy)
    (got,) = torch.autograd.grad(checkpoint(block, leaf, use_reentrant=False), leaf, gy)
    assert torch.equal(got, want)
    with torch.autograd.graph.save_on_cpu():
        y = block(leaf)
    assert torch.equal(torch.autograd.grad(y, leaf, gy)[0], want)
    y = block(leaf)
    with torch.no_grad():
        block.w_up.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, leaf, gy)
