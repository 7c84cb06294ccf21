"""Calls past what one launch takes."""
import pytest
import torch

from esr_amd import act8

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
