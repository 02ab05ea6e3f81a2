"""Arguments of the dense operators that are refused, on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_steps_are_whole_numbers():
    import numpy as np

    from cuda_mace_b200 import ops

    U = torch.randn(2, 20, 30, device="cuda")
    for steps in (2.5, 5.0, "5", None):
        with pytest.raises(TypeError):
            ops.orthogonalize(U, steps=steps)
    assert torch.equal(ops.orthogonalize(U, steps=np.int64(3)), ops.orthogonalize(U, steps=3))
