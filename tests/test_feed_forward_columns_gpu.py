"""Columns of the feed-forward block that differ in size, of x, of the weights and of the gradient: values that are 1e-8 of others in their block of
64 x 64 keep float32's precision.

Bounds as for rows, but that a block's values are off by at most 2^-49 of its largest: the low part of a pair is kept 2^11 times as large as the high
part's scale has it, fp16 values down to 2^-24 included, so a value of a block is off by 2^-22 of itself and by 2^-50 of the largest."""
import pytest
import torch

from tests.test_feed_forward_gpu import case
from tests.test_feed_forward_rows_gpu import inside, reference, run

pytestmark = pytest.mark.gpu

F32 = torch.float32
SIZES = [(300, 128, 512), (130, 136, 200), (9, 200, 130)]


def spread(n, least, dev):
    """n factors between `least` and 1, no two neighbours alike."""
    return (least ** ((torch.arange(n, device=dev, dtype=torch.float64) * 7 % 10) / 9))


@pytest.mark.parametrize("what", ["w_down", "hidden", "x", "grad", "w_gate"])
@pytest.mark.parametrize("least", [1e-3, 1e-5, 1e-8])
@pytest.mark.parametrize("M,C,H", SIZES)
def test_columns(M, C, H, least, what, dev="cuda"):
    args = [t.double() for t in case(M + 71, M, C, H, F32, dev)]
    x, wg, wu, wd, gy = args
    if what == "w_down":            # columns of y
        wd *= spread(C, least, dev)
    elif what == "hidden":          # hidden units whose values are small and whose rows of w_down bring them back
        f = spread(H, least, dev) ** 0.5
        wg, wu, wd = wg * f, wu * f, wd / (f * f)[:, None]
    elif what == "x":               # channels in other units, weights that fit them
        f = spread(C, least, dev)
        x, wg, wu = x * f, wg / f[:, None], wu / f[:, None]
    elif what == "grad":            # columns of the gradient of y
        gy = gy * spread(C, least, dev)
    else:
        wg = wg * spread(H, least, dev)
    args = [t.float() for t in (x, wg, wu, wd, gy)]
    inside(run(args), reference(*(t.double() for t in args), "silu", low=2.0 ** -11))
