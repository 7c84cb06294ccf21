"""The discriminator's layers as they are put together: upstream gradients of every layout, hooks, derivatives of every
order, 8-bit checkpoints against the definitions of gn_ref.py."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from esr_amd import bn  # noqa: E402

pytestmark = pytest.mark.gpu


def cl(t):
    return t.contiguous(memory_format=torch.channels_last)


def test_batch_norm_expanded_upstreams(gpu_device):
    """Upstream gradients of dγ and dβ that are expanded scalars (of a sum) give what whole tensors of them do."""
    torch.manual_seed(0)
    m = torch.nn.BatchNorm2d(24).to(gpu_device)
    x = cl(torch.randn(3, 24, 9, 7, device=gpu_device)).requires_grad_()
    gy = cl(torch.randn_like(x))
    gs = torch.autograd.grad(bn.bn_lrelu(x, m, 0.2), (x, m.weight, m.bias), gy, create_graph=True)
    up = [torch.full_like(g, s) for g, s in zip(gs, (0.5, 2.0, -3.0))]
    want = torch.autograd.grad(gs, (x, m.weight), up, retain_graph=True)
    got = torch.autograd.grad(0.5 * gs[0].sum() + 2.0 * gs[1].sum() - 3.0 * gs[2].sum(), (x, m.weight))
    for p, q in zip(got, want):
        assert torch.equal(p, q)
