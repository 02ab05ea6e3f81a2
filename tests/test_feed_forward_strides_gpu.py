"""Operands of the feed-forward block with strides of zero: expanded rows, weights and gradients, which sum what their positions get."""
import pytest
import torch

from tests.test_feed_forward_gpu import case, inside, reference

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "the gpu tests need a CUDA device"
    return torch.device("cuda:0")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,C,H", [(3, 24, 40), (70, 64, 96), (300, 136, 72)])
def test_expanded(M, C, H, dtype, dev):
    from cuda_mace_b200 import ops

    x, wg, wu, wd, gy = case(M + 61, M, C, H, dtype, dev)
    # one row for all positions, one row of gradients: values and gradients of contiguous copies, to the bit
    rows, grad = x[:1].expand(M, C), gy[:1].expand(M, C)
    assert rows.stride(0) == 0 and grad.stride(0) == 0

    def run(a, g):
        leaves = [t.detach().requires_grad_(True) for t in (a, wg, wu, wd)]
        y = ops.gated_feed_forward(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    got, want = run(rows, grad), run(rows.contiguous(), grad.contiguous())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    ref = reference(*(t.double() for t in (rows, wg, wu, wd, grad)), "silu", dtype)
    for name, a in zip(("y", "x", "w_gate", "w_up", "w_down"), got):
        inside(a, ref[name])
    # the gradient of the one row is the sum of its positions', each rounded to the type once, and the sum once more
    one = x[:1].clone().requires_grad_(True)
    y = ops.gated_feed_forward(one.expand(M, C), wg, wu, wd)
    (g,) = torch.autograd.grad(y, one, grad)
    v, bound = ref["x"]
    u = torch.finfo(dtype).eps / 2
    total = v.sum(0, keepdim=True)
    off = bound.sum(0, keepdim=True)
    assert ((g.double() - total).abs() <= off + (u + M * 2.0 ** -24) * (v.abs().sum(0, keepdim=True) + off)).all()
    # the gradient of a sum is expanded from one value
    (g,) = torch.autograd.grad(ops.gated_feed_forward(one.expand(M, C), wg, wu, wd).sum(), one)
    ones = reference(*(t.double() for t in (rows, wg, wu, wd, torch.ones_like(grad))), "silu", dtype)["x"]
    v, bound = ones
    total, off = v.sum(0, keepdim=True), bound.sum(0, keepdim=True)
    assert ((g.double() - total).abs() <= off + (u + M * 2.0 ** -24) * (v.abs().sum(0, keepdim=True) + off)).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_matrix_column_for_all(dtype, dev):
    """A weight that is one column expanded, and one that is a view of another's rows."""
    from cuda_mace_b200 import ops

    x, wg, wu, wd, gy = case(67, 90, 40, 56, dtype, dev)
    column = wg[:, :1]
    got = ops.gated_feed_forward(x, column.expand(40, 56), wu, wd)
    assert torch.equal(got, ops.gated_feed_forward(x, column.expand(40, 56).contiguous(), wu, wd))
    both = torch.cat([wg, wu], 1)
    assert torch.equal(ops.gated_feed_forward(x, both[:, :56], both[:, 56:], wd), ops.gated_feed_forward(x, wg, wu, wd))
