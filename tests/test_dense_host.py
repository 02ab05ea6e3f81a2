"""Argument checks of the dense operators that need no GPU: nothing is launched, nothing is written."""
import ctypes

import pytest
import torch

from cuda_mace_b200 import _abi, ops


def test_cpu_tensors_are_refused(built_library):
    x, w, wd = torch.zeros(3, 8), torch.zeros(8, 16), torch.zeros(16, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.gated_feed_forward(x, w, w, wd)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        ops.orthogonalize(w)
    with pytest.raises(ValueError, match="activation"):
        ops.gated_feed_forward(x, w, w, wd, activation="relu")


def test_workspace_queries(built_library):
    size = lambda *a: _abi.call("cmace_gated_ff_workspace_bytes", *a)  # noqa: E731
    assert size(1, 0, 64, 128, 0) > 0
    assert size(1, 1000, 64, 128, 1) > size(1, 1000, 64, 128, 0) > 0
    # float32: x, h and the weights as pairs of 16 bits, at least
    assert size(1, 4096, 64, 128, 0) >= 4 * (4096 * 64 + 4096 * 128 + 3 * 64 * 128)
    assert size(1, 1 << 30, 64, 128, 0) > 4 * (1 << 30) * 128      # 64-bit
    for bad in ((1, -1, 64, 128, 0), (1, 10, 0, 128, 0), (1, 10, 64, 0, 0), (1, 10, 1 << 21, 4, 0), (1, 1 << 31, 4, 4, 0)):
        assert size(*bad) == -1
    ortho = lambda *a: _abi.call("cmace_orthogonalize_workspace_bytes", *a)  # noqa: E731
    assert ortho(1, 4, 64, 64) > 0 and ortho(1, 0, 64, 64) > 0
    assert ortho(1, 2, 300, 500) >= 2 * 300 * 500 * 8
    for bad in ((1, -1, 8, 8), (1, 1, 0, 8), (1, 1, 8, 0), (1, 1, 1 << 21, 8)):
        assert ortho(*bad) == -1


def test_entries_refuse_before_they_launch(built_library):
    p = ctypes.c_void_p(256)   # never read: the checks come first
    for dtype in ("f32", "bf16"):
        fwd, bwd, ortho = (f"cmace_gated_ff_{d}_{dtype}" for d in ("fwd", "bwd")), None, f"cmace_orthogonalize_{dtype}"
        fwd, bwd = fwd
        with pytest.raises(RuntimeError, match="bad sizes"):
            _abi.call(fwd, p, p, p, p, -1, 8, 8, 0, p, p, 1 << 20, None, None)
        with pytest.raises(RuntimeError, match="activation"):
            _abi.call(fwd, p, p, p, p, 4, 8, 8, 2, p, p, 1 << 20, None, None)
        with pytest.raises(RuntimeError, match="null pointer"):
            _abi.call(fwd, p, None, p, p, 4, 8, 8, 0, p, p, 1 << 20, None, None)
        with pytest.raises(RuntimeError, match="needed"):
            _abi.call(fwd, p, p, p, p, 40, 8, 8, 0, p, p, 8, None, None)
        with pytest.raises(RuntimeError, match="aligned"):
            _abi.call(fwd, p, p, p, p, 40, 8, 8, 0, p, ctypes.c_void_p(264), 1 << 20, None, None)
        assert _abi.call(fwd, None, None, None, None, 0, 8, 8, 0, None, None, 0, None, None) == 0     # no rows: nothing to do
        with pytest.raises(RuntimeError, match="null pointer"):
            _abi.call(bwd, p, p, p, p, None, 4, 8, 8, 0, p, p, p, p, p, 1 << 20, None, None)
        assert _abi.call(bwd, p, p, p, p, p, 4, 8, 8, 0, None, None, None, None, None, 0, None, None) == 0   # no gradient wanted
        with pytest.raises(RuntimeError, match="bad sizes"):
            _abi.call(ortho, p, 1, 8, 8, 0, 1.0, 0.0, 0.0, 0.0, p, p, 1 << 20, None, None)
        with pytest.raises(RuntimeError, match="may grow"):
            _abi.call(ortho, p, 1, 8, 8, 50, 4.0, 0.0, 0.0, 0.0, p, p, 1 << 20, None, None)
        with pytest.raises(RuntimeError, match="null pointer"):
            _abi.call(ortho, p, 1, 8, 8, 5, 1.0, 0.0, 0.0, 0.0, None, p, 1 << 20, None, None)
        assert _abi.call(ortho, None, 0, 8, 8, 5, 1.0, 0.0, 0.0, 0.0, None, None, 0, None, None) == 0
