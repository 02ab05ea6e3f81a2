"""Codes that the dense operators' waits leave in the status word: one a wait, none of another operator's."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda_mace_b200", "csrc")
DENSE = ("tile_product.cuh", "gated_feed_forward.cu", "orthogonalize.cu")


def codes(name):
    with open(os.path.join(CSRC, name)) as f:
        return [int(c) for c in re.findall(r"(?:tp_report\(g|atomicCAS\([a-z.\->]*status, 0), (\d+)\)", f.read())]


def test_one_code_a_wait():
    dense = [c for name in DENSE for c in codes(name)]
    assert len(dense) >= 13 and len(set(dense)) == len(dense), sorted(dense)
    gemm = set(codes("gemm_tc.cu"))
    others = {c for name in os.listdir(CSRC) if name not in DENSE + ("gemm_tc.cu",) for c in codes(name)}
    assert not set(dense) & others and not set(dense) & gemm, (set(dense) & others, set(dense) & gemm)
