"""The number of kernels launched, as the binding counts them: what the operators launch, the backward in autograd's thread among it."""
import pytest
import torch

from tests.test_feed_forward_gpu import case

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def launches(f):
    from cuda_mace_b200 import _abi

    before = _abi.launch_count
    out = f()
    return _abi.launch_count - before, out


# forward: a pass over the weights 2, the whole block 1, rows and weights laid out 1 (2 with sizes of wide rows) and two products, bf16 where it lies 2;
# backward: layout as for the forward pass (bf16: 0), hidden values, gradient of x, two products or one and a sum for the weights
@pytest.mark.parametrize("M,C,H,dtype,forward,backward", [(4, 512, 1024, F32, 2, None), (100, 64, 128, F32, 1, None), (9000, 64, 128, F32, 3, 5),
                                                          (9000, 192, 256, F32, 4, 6), (9000, 64, 128, BF16, 2, 4), (9000, 65, 128, BF16, 3, 5)])
def test_feed_forward(M, C, H, dtype, forward, backward):
    from cuda_mace_b200 import ops

    x, wg, wu, wd, gy = case(3, M, C, H, dtype, "cuda")
    n, _ = launches(lambda: ops.gated_feed_forward(x, wg, wu, wd))
    assert n == forward
    if backward:
        leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
        y = ops.gated_feed_forward(*leaves)
        n, _ = launches(lambda: torch.autograd.grad(y, leaves, gy))
        assert n == backward


@pytest.mark.parametrize("shape,steps,count", [((3, 64, 64), 5, 1), ((0, 64, 64), 5, 0), ((1, 140, 200), 3, 2 + 9)])
def test_orthogonalize(shape, steps, count):
    from cuda_mace_b200 import ops

    U = torch.randn(*shape, device="cuda")
    assert launches(lambda: ops.orthogonalize(U, steps=steps))[0] == count


def test_no_rows():
    from cuda_mace_b200 import ops

    x, wg, wu, wd, _ = case(3, 1, 64, 128, F32, "cuda")
    assert launches(lambda: ops.gated_feed_forward(x[:0], wg, wu, wd))[0] == 0
