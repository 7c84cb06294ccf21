"""Group norm and 8-bit activation checkpoints without a GPU: the closed forms the GPU tests compare with against
autograd and differences, the refusals of the Python and C entry points, and the discriminator's options."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import gn_ref as R  # noqa: E402
from esr_amd import _lib, act8, dconv, gn, networks  # noqa: E402
from esr_amd.discriminator import Discriminator_VGG_128_  # noqa: E402


@pytest.mark.parametrize('shape,G', [((2, 6, 3, 5), 3), ((1, 4, 2, 2), 1), ((3, 5, 4, 3), 5)])
def test_closed_forms_match_autograd(shape, G):
    c = R.case(shape, G, seed=3)
    f = R.forward(c)
    x, w, b, gy = (torch.from_numpy(v).requires_grad_() for v in (c.x, c.w, c.b, c.gy))
    z = torch.nn.functional.group_norm(x, G, w, b, c.eps)
    y = torch.where(z > 0, z, c.slope * z)
    np.testing.assert_allclose(f.y, y.detach().numpy(), rtol=1e-12, atol=1e-13)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
    d = R.backward(c, f)
    for mine, ref in ((d.gx, gx), (d.gw, gw), (d.gb, gb)):
        np.testing.assert_allclose(mine, ref.detach().numpy(), rtol=1e-9, atol=1e-11)
    L = (gx * torch.from_numpy(c.u)).sum() + (gw * torch.from_numpy(c.ga)).sum() + (gb * torch.from_numpy(c.gb)).sum()
    g2 = torch.autograd.grad(L, (x, gy, w))
    e = R.backward2(c, f, d)
    for mine, ref in zip((e.g_x, e.g_gy, e.g_w), g2):
        np.testing.assert_allclose(mine, ref.numpy(), rtol=1e-8, atol=1e-10)


def test_backward_matches_differences():
    c = R.case((2, 6, 4, 5), 2, seed=9)
    d = R.backward(c, R.forward(c))
    rng = np.random.default_rng(1)
    for name, g in (('x', d.gx), ('w', d.gw), ('b', d.gb)):
        v = rng.standard_normal(g.shape)
        base, t = getattr(c, name), 1e-6
        loss = []
        for s in (t, -t):
            setattr(c, name, base + s * v)
            loss.append((R.forward(c).y * c.gy).sum())
        setattr(c, name, base)
        # central differences: t² third derivatives plus 1e-16 / t rounding of the loss
        np.testing.assert_allclose((loss[0] - loss[1]) / (2 * t), (g * v).sum(), rtol=1e-6, atol=1e-7)


def test_block_reference():
    """The 8-bit reference itself: error at most half a step (a step for positive values that would round to 0), the
    largest magnitude in range, exact powers of two at the range's ends."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 70)) * np.exp2(rng.integers(-60, 60, (50, 1)))).astype(np.float32)
    codes, exps, v = R.pack(x)
    step = np.exp2(exps.astype(np.float64) - 132).repeat(32, 1)[:, :70]
    assert np.abs(codes).max() == 127 and codes.min() >= -127
    tiny = (x > 0) & (x < step / 2)
    assert (np.abs(v - x)[~tiny] <= step[~tiny] / 2).all() and (v[tiny] == step[tiny]).all()
    assert ((v > 0) == (x > 0)).all()
    top = np.abs(np.pad(x, ((0, 0), (0, 26))).reshape(50, 3, 32)).max(2)
    s = np.exp2(exps.astype(np.float64) - 132)
    assert (127 * s >= top).all() and (127 * s / 2 < top).all()


def test_refusals():
    x = torch.zeros(2, 8, 4, 4)
    for bad in (lambda: gn.group_norm_lrelu(x, 3), lambda: gn.group_norm_lrelu(x, 0),
                lambda: gn.group_norm_lrelu(x[0], 2), lambda: gn.group_norm_lrelu(x, 2, checkpoint='int4'),
                lambda: gn.group_norm_lrelu(x, 2, torch.zeros(7)), lambda: gn.group_norm_lrelu(x, 2, eps=-1.0),
                lambda: gn.group_norm_lrelu(x, 2, slope=math.inf), lambda: gn.group_norm_lrelu(x[:, :, :0], 2),
                lambda: gn.HipGroupNorm(2, 8, checkpoint='fp8'), lambda: gn.HipGroupNorm(3, 8)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: gn.group_norm_lrelu(x, 2), lambda: gn.HipGroupNorm(2, 8)(x), lambda: act8.pack(x),
                lambda: act8.Act8(torch.zeros(2, 48, dtype=torch.int8), torch.zeros(2, 2, dtype=torch.uint8), 40).unpack()):
        with pytest.raises(RuntimeError, match='ROCm device'):
            bad()
    i8, u8 = (lambda *s: torch.zeros(*s, dtype=torch.int8)), (lambda *s: torch.zeros(*s, dtype=torch.uint8))
    for bad in ((i8(2, 48), u8(2, 1), 40), (torch.zeros(2, 48), u8(2, 2), 40), (i8(2, 40), u8(2, 2), 40),
                (i8(2, 48), i8(2, 2), 40), (i8(2, 48), u8(2, 2), 49), (i8(2, 0), u8(2, 0), 0)):
        with pytest.raises(ValueError):
            act8.Act8(*bad)
    with pytest.raises(RuntimeError, match='ROCm device'):
        dconv.conv_wgrad_act8(act8.Act8(i8(1, 4, 4, 16), u8(1, 4, 4, 1), 8), torch.zeros(1, 4, 4, 8), 3, 1, 1)
    conv = dconv.HipConv2d(8, 8, 3, padding=1)
    conv.act_checkpoint = 'int4'
    with pytest.raises(ValueError):
        conv.keeps8()


def test_c_entries_refuse():
    """Every check of the C entries comes before any launch: bad sizes and pointers return ESR_EINVAL."""
    lib = _lib.load()
    p = 1 << 20  # never dereferenced
    E = -1
    assert lib.esr_act8_pack(None, 1, 1, p, p, None) == E and lib.esr_act8_pack(p, 0, 4, p, p, None) == E
    assert lib.esr_act8_unpack(p, None, 1, 1, p, None) == E and lib.esr_act8_unpack(p, p, 1, 0, p, None) == E
    assert lib.esr_act8_pack(p, 1 << 45, 64, p, p, None) == E
    assert lib.esr_act8_pack(p, 1, 1, p + 4, p, None) == E and lib.esr_act8_unpack(p + 8, p, 1, 1, p, None) == E  # alignment
    ok = (2, 16, 8, 4)
    assert lib.esr_gn_workspace_bytes(*ok) > 0
    for bad in ((0, 16, 8, 4), (2, 0, 8, 4), (2, 16, 8, 3), (2, 16, 0, 1), (2, 16, 8, 0), (70000, 16, 8, 4),
                (2, 1 << 40, 64, 4)):
        assert lib.esr_gn_workspace_bytes(*bad) == E
        assert lib.esr_gn_lrelu_fwd(p, *bad, None, None, 1e-5, 0.2, p, p, None, None, None, None, p, None) == E
    assert lib.esr_gn_lrelu_fwd(p, *ok, None, None, -1.0, 0.2, p, p, None, None, None, None, p, None) == E
    for blocks in ((p, None, None, None), (None, None, None, p)):  # codes without exponents
        assert lib.esr_gn_lrelu_fwd(p, *ok, None, None, 1e-5, 0.2, p, p, *blocks, p, None) == E
    assert lib.esr_gn_lrelu_bwd(p, None, None, p, *ok, None, None, p, 0.2, None, p, p, p, p, None) == E
    bwd = lambda x, c, e: lib.esr_gn_lrelu_bwd(x, c, e, p, *ok, None, None, p, 0.2, p, p, p, p, p, None)  # noqa: E731
    assert bwd(None, p + 4, p) == E and bwd(None, None, None) == E and bwd(p, p, p) == E and bwd(None, p, None) == E
    assert lib.esr_gn_lrelu_bwd2(None, p, p, p, None, None, None, *ok, None, None, p, 0.2, None, p, p, p, p, None) == E
    geo = (2, 8, 8, 64, 8, 8, 64, 3, 1, 1)
    n = lib.esr_dconv_wgrad_act8_workspace_bytes(*geo)
    assert n > 0
    for i, v in ((0, 0), (4, 7), (5, 9), (7, 9), (7, 0), (8, 0), (9, -1), (3, 0), (6, 0)):
        bad = list(geo)
        bad[i] = v
        assert lib.esr_dconv_wgrad_act8_workspace_bytes(*bad) == E, (i, v)
        assert lib.esr_dconv_wgrad_act8(p, p, *bad[:4], p, *bad[4:], p, p, None) == E, (i, v)
    assert lib.esr_dconv_wgrad_act8(p, None, *geo[:4], p, *geo[4:], p, p, None) == E
    assert lib.esr_dconv_wgrad_act8(p + 4, p, *geo[:4], p, *geo[4:], p, p, None) == E


def _opt(**d):
    return {'gpu_ids': None, 'datasets': {'train': {'patch_size': 96}},
            'network_D': dict({'which_model_D': 'discriminator_vgg_128', 'in_nc': 3, 'nf': 64, 'norm_type': 'batch',
                               'act_type': 'leakyrelu', 'mode': 'CNA', 'n_layers': 6}, **d)}


def test_discriminator_options():
    keys = lambda **d: list(networks.define_D(_opt(**d)).state_dict())  # noqa: E731
    batch, group, inst = keys(), keys(norm_type='group'), keys(norm_type='instance')
    assert any('running_mean' in k for k in batch) and not any('running' in k for k in group + inst)
    assert [k for k in batch if 'running' not in k and 'num_batches' not in k and 'classifier.2.1' not in k] == group
    assert len(inst) == len(group) - 2 * 6  # no affine parameters
    netD = networks.define_D(_opt(norm_type='group', norm_groups=16, act_checkpoint='int8'))
    norms = [m for m in netD.modules() if isinstance(m, gn.HipGroupNorm)]
    assert [m.num_groups for m in norms] == [16] * 5 + [4] and all(m.checkpoint == 'int8' for m in norms)
    convs = [m for m in netD.modules() if isinstance(m, dconv.HipConv2d)]
    assert len(convs) == 8 and all(m.act_checkpoint == 'int8' for m in convs)
    assert all(m.act_checkpoint is None for m in networks.define_D(_opt()).modules() if isinstance(m, dconv.HipConv2d))
    for bad, err in (({'norm_type': 'layer'}, NotImplementedError), ({'norm_groups': 0}, ValueError),
                     ({'act_checkpoint': 'fp4'}, ValueError)):
        with pytest.raises(err):
            networks.define_D(_opt(**bad))


def test_ddp_without_buffers(monkeypatch):
    """A discriminator with group norm has no buffers: the per-step broadcast of rank 0's is nothing."""
    from esr_amd import SRRaGAN_model as S
    netD = Discriminator_VGG_128_(3, 64, norm_type='group', nb=2)
    calls = []
    monkeypatch.setattr(S, '_world', lambda: 2)
    monkeypatch.setattr(S, 'collective', lambda *a, **k: calls.append(a))
    flat = S.FlatBuffers(netD)
    assert flat.sync() is None
    S._broadcast_buffers(netD, flat)
    S._broadcast_buffers(netD)
    assert not calls
