"""Arguments of the dense operators that are refused, on the device."""
import pytest
import torch

from tests.test_feed_forward_gpu import case

pytestmark = pytest.mark.gpu


def test_steps_are_whole_numbers():
    import numpy as np

    from cuda_mace_b200 import ops

    U = torch.randn(2, 20, 30, device="cuda")
    for steps in (2.5, 5.0, "5", None):
        with pytest.raises(TypeError):
            ops.orthogonalize(U, steps=steps)
    assert torch.equal(ops.orthogonalize(U, steps=np.int64(3)), ops.orthogonalize(U, steps=3))


def test_status_of_the_torch_operator():
    from cuda_mace_b200 import ops

    args = case(5, 20, 16, 24, torch.float32, "cuda")[:4]
    want = ops.gated_feed_forward(*args)   # loads the library
    op = torch.ops.cmace_b200.gated_feed_forward
    assert torch.equal(op(*args, 0, torch.zeros(1, dtype=torch.int32, device="cuda")), want)
    for status in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")):
        with pytest.raises(RuntimeError, match="status"):
            op(*args, 0, status)
    with pytest.raises(RuntimeError, match="activation"):
        op(*args, 7, torch.zeros(1, dtype=torch.int32, device="cuda"))
