"""Calls past what one launch takes, and launches of few large parts."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from esr_amd import act8  # noqa: E402
from test_gpu_act8 import check_wgrad, wgrad_case  # noqa: E402

pytestmark = pytest.mark.gpu


def test_pack_more_rows_than_a_grid(gpu_device):
    """2^29 rows and some of one channel (a workgroup takes 32 rows, a grid 2^24 workgroups of 256 threads): rows around the
    borders of the launches and the last ones are those of a short call."""
    n = 2 ** 29 + 77
    x = torch.randn(n, 1, device=gpu_device)
    q = act8.pack(x)
    v = q.unpack()
    for at in (0, 2 ** 28 - 40, 2 ** 28, 2 ** 29 - 40, 2 ** 29, n - 50):
        s = slice(at, at + 50)
        want = act8.pack(x[s].clone())
        assert torch.equal(q.codes[s], want.codes) and torch.equal(q.exps[s], want.exps), at
        assert torch.equal(v[s], want.unpack()), at
    assert bool(((v - x).abs() <= x.abs() / 127).all())  # half a step of a block of one value


# many 64 x 64 weights and few pixels: fewer than eight splits, and numbers of them that eight does not divide
@pytest.mark.parametrize('geo', [(1, 9, 9, 512, 320, 8, 1, 0), (5, 11, 13, 320, 100, 8, 1, 0), (3, 10, 9, 256, 512, 3, 1, 1),
                                 (2, 9, 33, 448, 320, 4, 2, 1), (1, 5, 6, 512, 448, 5, 1, 2), (7, 17, 18, 128, 192, 3, 1, 1)])
def test_weight_gradient_of_few_splits(gpu_device, geo):
    x, gy = wgrad_case(geo, sum(geo))
    check_wgrad(gpu_device, x, gy, *geo[5:])
