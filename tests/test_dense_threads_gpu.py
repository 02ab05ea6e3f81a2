"""First calls of the dense operators from several threads at once, each in a process of its own where nothing has been set up."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# Updates of one kernel that ask for different amounts of shared memory: 64 and 128 columns, 150 and 250 (of a stack that fills the SMs)
PROGRAM = """
import threading
import torch
from cuda_mace_b200 import _abi, ops

sets = [torch.randn(*s, device="cuda") for s in ((1, 64, 64), (1, 128, 128), (1, 32, 150), (80, 32, 250))]
for U in sets:
    ops._orthogonalize_bytes(True, *U.shape)   # no launch
ws = [torch.empty(256, dtype=torch.uint8, device="cuda") for _ in sets]
outs = [torch.empty_like(U) for U in sets]
_abi.load()
torch.cuda.synchronize()
failed = []
for pair in ((0, 1), (2, 3)):
    gate = threading.Barrier(len(pair))

    def run(k):
        torch.cuda.set_device(0)
        args = (sets[k].data_ptr(), *sets[k].shape, 5, 3.4445, -4.7750, 2.0315, 1e-7, outs[k].data_ptr(), ws[k].data_ptr(), 256, 0, 0)
        gate.wait()
        try:
            _abi.call("cmace_orthogonalize_f32", *args)
        except RuntimeError as e:
            failed.append(str(e))

    threads = [threading.Thread(target=run, args=(k,)) for k in pair]
    [t.start() for t in threads]
    [t.join() for t in threads]
torch.cuda.synchronize()
assert not failed, failed
for U, out in zip(sets, outs):
    assert torch.equal(out, ops.orthogonalize(U))
"""


@pytest.mark.parametrize("run", range(3))
def test_first_calls_of_two_threads(run):
    r = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-2000:]
