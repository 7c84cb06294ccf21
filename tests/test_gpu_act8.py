"""Activations kept in 8 bits (esr_amd/act8.py) and the convolution weight gradient that reads them, against the
definitions of gn_ref.py."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import gn_ref as R  # noqa: E402
from esr_amd import act8, dconv, gn, networks  # noqa: E402
from esr_amd.discriminator import Discriminator_VGG_128_  # noqa: E402
from esr_amd.loss import GradientPenaltyLoss  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('P,C', [(1, 1), (1, 32), (3, 31), (2, 33), (7, 100), (1000, 64), (257, 4), (65, 130), (5, 515),
                                 (4099, 37)])
def test_pack_is_the_definition(gpu_device, P, C):
    rng = np.random.default_rng(P + C)
    x = (rng.standard_normal((P, C)) * np.exp2(rng.integers(-20, 20, (P, 1)))).astype(np.float32)
    codes, exps, v = R.pack(x)
    q = act8.pack(torch.from_numpy(x).to(gpu_device))
    got = q.codes.cpu().numpy()
    assert np.array_equal(got[:, :C], codes) and not got[:, C:].any() and np.array_equal(q.exps.cpu().numpy(), exps)
    assert np.array_equal(q.unpack().cpu().numpy(), v.astype(np.float32))
    assert q.nbytes == P * (-(-C // 16) * 16 + -(-C // 32)) and q.shape == (P, C)


def test_pack_extremes(gpu_device):
    """Zeros, subnormals, the largest floats, ties, infinities and NaN; every block on its own."""
    f = np.float32
    x = np.zeros((12, 32), dtype=f)
    x[1, 3] = np.finfo(f).max
    x[2] = np.finfo(f).smallest_subnormal
    x[3, :2] = [np.finfo(f).tiny, -np.finfo(f).tiny / 4]
    x[4, 0] = np.inf
    x[5, 31] = -np.inf
    x[6, 7] = np.nan
    x[7] = np.arange(32) + 0.5  # ties at step 1/4, 1/2 ...
    x[7, 0] = 127
    x[8] = np.linspace(-1e-3, 1e-3, 32)
    x[8, 0] = 1.0
    x[9, 0], x[9, 1] = f(127 / 64), np.nextafter(f(127 / 64), f(2))
    x[10, 0] = f(127 / 64)
    x[11, :3] = [-5.0, -0.0, 2.0 ** -140]
    codes, exps, v = R.pack(x)
    q = act8.pack(torch.from_numpy(x).to(gpu_device))
    assert np.array_equal(q.exps.cpu().numpy(), exps) and np.array_equal(q.codes.cpu().numpy(), codes)
    np.testing.assert_array_equal(q.unpack().cpu().numpy(), v.astype(f))
    assert np.isfinite(v[1]).all()


def test_pack_layouts(gpu_device):
    x = torch.randn(3, 5, 7, 40, device=gpu_device)
    want = act8.pack(x)
    off = torch.empty(x.numel() + 1, device=gpu_device)[1:].view(x.shape).copy_(x)
    wide = torch.randn(3, 5, 7, 60, device=gpu_device)
    wide[..., 11:51] = x
    for v in (off, wide[..., 11:51], x.transpose(1, 2).contiguous().transpose(1, 2)):
        q = act8.pack(v)
        assert torch.equal(q.codes, want.codes) and torch.equal(q.exps, want.exps)
    assert act8.pack(x[:0]).unpack().shape == (0, 5, 7, 40)
    codes = torch.empty(want.codes.numel() + 1, device=gpu_device, dtype=torch.int8)[1:].view(want.codes.shape)
    assert torch.equal(act8.Act8(codes.copy_(want.codes), want.exps, 40).unpack(), want.unpack())


# B, H, W, Ci, Co, k, s, p: every layer kind of the discriminator, ragged channels, maps smaller than the kernel's reach,
# one output, strides that leave a border unread, many images of few pixels
GEO = [(1, 1, 1, 1, 1, 1, 1, 0), (2, 5, 7, 3, 2, 3, 1, 1), (1, 12, 10, 64, 64, 3, 1, 1), (2, 9, 13, 64, 128, 3, 1, 1),
       (2, 16, 20, 64, 64, 4, 2, 1), (1, 15, 17, 33, 70, 4, 2, 1), (1, 9, 9, 128, 96, 4, 1, 1), (2, 11, 9, 40, 100, 8, 1, 0),
       (3, 8, 8, 256, 100, 8, 1, 0), (4, 6, 5, 100, 1, 1, 1, 0), (1, 2, 3, 65, 64, 3, 1, 1), (1, 40, 70, 32, 64, 3, 1, 1),
       (37, 3, 3, 64, 64, 3, 1, 1), (1, 7, 200, 96, 32, 3, 2, 1), (2, 10, 11, 16, 16, 5, 3, 2), (1, 6, 6, 8, 8, 2, 1, 0),
       (1, 33, 34, 64, 64, 7, 1, 3), (2, 4, 300, 64, 64, 1, 1, 0), (1, 3, 3, 8, 8, 3, 1, 5), (1, 90, 67, 64, 64, 3, 1, 1)]


def wgrad_case(geo, seed, dist=1.0):
    B, H, W, Ci, Co, k, s, p = geo
    r = np.random.default_rng(seed)
    x = r.standard_normal((B, H, W, Ci)) * np.exp2(dist * r.standard_normal((B, H, W, 1)))
    x = np.where(x > 0, x, 0.2 * x).astype(np.float32)
    gy = r.standard_normal((B, dconv.out_size(H, k, s, p), dconv.out_size(W, k, s, p), Co)).astype(np.float32)
    return x, gy


def check_wgrad(g, x, gy, k, s, p):
    v = R.pack(x.reshape(-1, x.shape[3]))[2].reshape(x.shape)
    ref, mag = R.wgrad(v, gy, k, s, p)
    got = dconv.conv_wgrad_act8(act8.pack(torch.from_numpy(x).to(g)), torch.from_numpy(gy).to(g), k, s, p)
    assert got.shape == ref.shape
    got = got.double().cpu().numpy()
    K = gy[..., 0].size
    # gy's two pieces keep 2^-21 of it (and 2^-38 of its largest value); K float32 additions round by 2^-24 of a partial
    # sum each: sqrt(K) of them in the mean, K at worst
    tiny = 2.0 ** -38 * np.abs(gy).max(initial=0) * np.abs(v).sum((0, 1, 2)).reshape(1, -1, 1, 1)
    assert (np.abs(got - ref) <= (2.0 ** -21 + K * R.U) * mag + tiny).all()
    n = np.linalg.norm
    assert n(got - ref) <= (2.0 ** -21 + 2 * np.sqrt(K) * R.U) * n(mag) + 1e-30
    return got


@pytest.mark.parametrize('geo', GEO)
def test_wgrad_against_definition(gpu_device, geo):
    x, gy = wgrad_case(geo, sum(geo))
    check_wgrad(gpu_device, x, gy, *geo[5:])


@pytest.mark.parametrize('kind', ['tiny_gy', 'huge_gy', 'growing_gy', 'zeros', 'tiny_x', 'wide_x'])
def test_wgrad_ranges(gpu_device, kind):
    """Gradients far from 1, growing by 2^60 over the pixels, zero tiles first; activations of very different pixels."""
    geo = (2, 24, 40, 64, 64, 3, 1, 1)
    x, gy = wgrad_case(geo, 3, 6.0 if kind == 'wide_x' else 1.0)
    if kind == 'tiny_gy':
        gy *= np.float32(1e-20)
    elif kind == 'huge_gy':
        gy *= np.float32(1e15)
    elif kind == 'growing_gy':
        gy *= np.exp2(np.linspace(-30, 30, 2 * 24)).reshape(2, 24, 1, 1).astype(np.float32)
    elif kind == 'zeros':
        gy[0] = 0
        x[0, :12] = 0
    elif kind == 'tiny_x':
        x *= np.float32(1e-25)
    check_wgrad(gpu_device, x, gy, 3, 1, 1)


@pytest.mark.parametrize('below', [0, 11, 16, 20, 24, 27])
def test_wgrad_of_blocks_far_below_the_largest(gpu_device, below):
    """A block's codes are exact down to 2^-27 of the workgroup's largest: where only that block's pixel has a gradient,
    the weights are its values times the gradient."""
    x = np.zeros((1, 1, 2, 32), np.float32)
    x[0, 0, 0] = np.arange(32) * 4 + 3
    x[0, 0, 1] = (np.arange(32) * 4 + 3) * np.float32(2.0 ** -below)
    gy = np.zeros((1, 1, 2, 64), np.float32)
    gy[0, 0, 1] = np.linspace(-1.3, 1.7, 64)
    got = dconv.conv_wgrad_act8(act8.pack(torch.from_numpy(x).to(gpu_device)), torch.from_numpy(gy).to(gpu_device), 1, 1,
                                0).double().cpu().numpy()[:, :, 0, 0]
    want = np.outer(gy[0, 0, 1].astype(np.float64), x[0, 0, 1].astype(np.float64))
    # The gradient's two pieces (2^-22 of it + 2^-36 of the largest, 2) and two additions' roundings.  Those of an x that
    # is a subnormal f16 are 2^-24 of the product that f16's least exponent gives: x is staged at 8 times its value here
    # (step 1, scale 2^3), so of 2^-13 / 8 times the gradient's next power of two, twice: 2 · 2^-24 · 2^-16 · 2 |gy|.
    sub = 2.0 ** -38 * np.abs(gy[0, 0, 1].astype(np.float64))[:, None]
    assert (np.abs(got - want) <= 2.0 ** -21 * np.abs(want) + 2.0 ** -35 * np.abs(x[0, 0, 1]) + sub).all()


@pytest.mark.parametrize('where', ['x', 'gy'])
def test_wgrad_nonfinite(gpu_device, where):
    """A NaN reaches the weights that it belongs to: its block's input channels, or its output channel."""
    geo = (1, 10, 9, 64, 70, 3, 1, 1)
    x, gy = wgrad_case(geo, 4)
    if where == 'x':
        x[0, 4, 4, 40] = np.nan
    else:
        gy[0, 5, 5, 65] = np.inf
    got = dconv.conv_wgrad_act8(act8.pack(torch.from_numpy(x).to(gpu_device)), torch.from_numpy(gy).to(gpu_device), 3,
                                1, 1).cpu().numpy()
    bad = ~np.isfinite(got)
    if where == 'x':
        assert bad[:, 32:].all() and not bad[:, :32].any()
    else:
        assert bad[65].all() and not bad[:65].any() and not bad[66:].any()


@pytest.mark.parametrize('geo', [(1, 8, 9, 32, 64, 3, 2, 0), (2, 7, 9, 64, 40, 4, 2, 0), (1, 12, 30, 33, 8, 2, 5, 0),
                                 (1, 3, 3, 8, 8, 1, 100, 5)])
def test_wgrad_of_pixels_that_no_output_reads(gpu_device, geo):
    """Infinities in rows and columns that the strides leave unread do not reach the weights."""
    B, H, W, Ci, Co, k, s, p = geo
    x, gy = wgrad_case(geo, 9)
    want = check_wgrad(gpu_device, x, gy, k, s, p)
    rows, cols = (max(0, (dconv.out_size(n, k, s, p) - 1) * s + k - p) for n in (H, W))
    assert rows < H or cols < W
    x[:, rows:], x[:, :, cols:] = np.inf, np.nan
    got = dconv.conv_wgrad_act8(act8.pack(torch.from_numpy(x).to(gpu_device)), torch.from_numpy(gy).to(gpu_device), k, s, p)
    assert np.array_equal(got.double().cpu().numpy(), want)


def test_wgrad_refusals(gpu_device):
    x8 = act8.pack(torch.randn(2, 6, 6, 8, device=gpu_device))
    gy = torch.randn(2, 6, 6, 16, device=gpu_device)
    assert dconv.conv_wgrad_act8(x8, gy, 3, 1, 1).shape == (16, 8, 3, 3)
    for bad in ((gy, 3, 1, 0), (gy, 3, 2, 1), (gy, 9, 1, 4), (gy, 0, 1, 1), (gy[:1], 3, 1, 1), (gy[0], 3, 1, 1),
                (gy, 3, 0, 1)):
        with pytest.raises(ValueError):
            dconv.conv_wgrad_act8(x8, *bad)
    with pytest.raises(RuntimeError, match='float32'):
        dconv.conv_wgrad_act8(x8, gy.half(), 3, 1, 1)
    empty = act8.pack(torch.randn(0, 6, 6, 8, device=gpu_device))
    assert float(dconv.conv_wgrad_act8(empty, gy[:0], 3, 1, 1).abs().sum()) == 0


def test_wgrad_strided_gradient_and_determinism(gpu_device):
    x = torch.randn(2, 30, 31, 64, device=gpu_device)
    x8 = act8.pack(x)
    gy = torch.randn(2, 64, 30, 31, device=gpu_device).permute(0, 2, 3, 1)
    want = dconv.conv_wgrad_act8(x8, gy, 3, 1, 1)
    off = torch.empty(gy.numel() + 1, device=gpu_device)[1:].view(gy.shape).copy_(gy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(s):
            a = dconv.conv_wgrad_act8(x8, gy, 3, 1, 1)
        b = dconv.conv_wgrad_act8(x8, off, 3, 1, 1)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)


@pytest.mark.parametrize('k,s,p', [(3, 1, 1), (4, 2, 1), (1, 1, 0)])
def test_conv_layer_checkpoint(gpu_device, k, s, p):
    """HipConv2d with act_checkpoint: output, data gradient and bias gradient bit for bit those of the plain layer, the
    weight gradient that of the blocks' values, and the double backward's terms."""
    torch.manual_seed(k)
    convs = []
    for ck in (None, 'int8'):
        m = dconv.HipConv2d(64, 32, k, stride=s, padding=p).to(gpu_device)
        m.act_checkpoint = ck
        convs.append(m)
    convs[1].load_state_dict(convs[0].state_dict())
    x = torch.randn(2, 64, 14, 18, device=gpu_device).contiguous(memory_format=torch.channels_last)
    xv = act8.pack(x.permute(0, 2, 3, 1)).unpack().permute(0, 3, 1, 2)
    gy = torch.randn_like(convs[0](x)).requires_grad_()
    u, V, t = torch.randn_like(x), torch.randn_like(convs[0].weight), torch.randn(32, device=gpu_device)
    res = []
    for m, inp in ((convs[0], x), (convs[1], x), (convs[0], xv)):
        inp = inp.detach().requires_grad_()
        y = m(inp)
        gx, gw, gb = torch.autograd.grad(y, (inp, m.weight, m.bias), gy, create_graph=True)
        L = (gx * u).sum() + (gw * V).sum() + (gb * t).sum()
        res.append([y, gx, gw, gb] + list(torch.autograd.grad(L, (inp, gy, m.weight))))
    plain, ck, at = res
    for i in (0, 1, 3, 4, 6):  # y, gx, gb, and the second-order terms that do not hold x
        assert torch.equal(plain[i], ck[i]), i
    for i in (2, 5):  # gw and its term in g_gy: of the blocks' values
        assert float((ck[i] - at[i]).norm() / at[i].norm()) < 2e-6, i
    # first-order only, without a graph; a frozen layer keeps nothing
    y = convs[1](x)
    gw, = torch.autograd.grad(y, convs[1].weight, gy.detach())
    assert torch.equal(gw, ck[2])
    convs[1].weight.requires_grad_(False)
    assert not convs[1].keeps8()
    with pytest.raises(ValueError):
        convs[1].weight.requires_grad_(True)
        convs[1](x, act8.pack(torch.zeros(1, 2, 2, 64, device=gpu_device)))


def test_conv_layer_graph_capture(gpu_device):
    """A checkpointed layer's forward, backward and double backward captured once, replayed between eager calls."""
    m = dconv.HipConv2d(64, 32, 3, padding=1).to(gpu_device)
    m.act_checkpoint = 'int8'
    w0, b0 = m.weight.detach(), m.bias.detach()
    shape = (2, 64, 12, 14)
    mk = lambda c: torch.randn(2, c, 12, 14, device=gpu_device).contiguous(  # noqa: E731
        memory_format=torch.channels_last)
    static = [mk(64), mk(32), mk(64)]

    def step(x, gy, u):
        x, gy = x.detach().requires_grad_(), gy.detach().requires_grad_()
        w, b = w0.detach().requires_grad_(), b0.detach().requires_grad_()
        xh = x.permute(0, 2, 3, 1)
        x8 = act8.pack(xh)
        y = dconv.DConvAct8Fn.apply(xh, act8.Carrier.apply(xh), x8.codes, x8.exps, w, b, 3, 1, 1).permute(0, 3, 1, 2)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
        return (y.detach(), gx.detach(), gw.detach()) + torch.autograd.grad((gx * u).sum() + gw.sum(), (x, gy, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for k in range(3):
        new = [mk(64) * (k + 1), mk(32), mk(64)]
        want = step(*new)
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for i, (p, q) in enumerate(zip(out, want)):
            assert torch.equal(p, q), (i, shape)


def test_offsets_past_31_bits(gpu_device):
    """More than 2^31 values: the last ones are packed, read, normalised and multiplied like the first."""
    x = torch.randn(3, 3400, 3400, 64, device=gpu_device)
    assert x.numel() > 2 ** 31
    q = act8.pack(x)
    last = act8.pack(x[2, -5:])
    assert torch.equal(q.codes[2, -5:], last.codes) and torch.equal(q.exps[2, -5:], last.exps)
    assert torch.equal(act8.Act8(q.codes[2, -5:], q.exps[2, -5:], 64).unpack(), last.unpack())
    v = q.unpack()
    assert torch.equal(v[2, -5:], last.unpack())
    del v
    with torch.no_grad():
        y = gn.group_norm_lrelu(x.permute(0, 3, 1, 2), 32)[2, :, -4:].clone()
        y1 = gn.group_norm_lrelu(x[2:].permute(0, 3, 1, 2), 32)[0, :, -4:]
    torch.testing.assert_close(y, y1, rtol=2 ** -22, atol=1e-9)  # the sums' order differs: 1e-16 of the statistics
    del x
    gy = torch.randn(3, 3400, 3400, 4, device=gpu_device)
    whole = dconv.conv_wgrad_act8(q, gy, 1, 1, 0)
    parts = sum(dconv.conv_wgrad_act8(act8.Act8(q.codes[i:i + 1], q.exps[i:i + 1], 64), gy[i:i + 1], 1, 1, 0).double()
                for i in range(3))
    # sums of 3.5e7 products in float32, of order sqrt(3.5e7): 2^-24 of a partial sum per addition of a 256-way split
    torch.testing.assert_close(whole.double(), parts, rtol=0, atol=2 ** -24 * (3.5e7 / 256) ** 0.5 * 5900)


def _disc(g, norm, ck, seed=0):
    torch.manual_seed(seed)
    netD = Discriminator_VGG_128_(3, 64, norm_type=norm, nb=6, num_2_strides=3, act_checkpoint=ck)
    networks.init_weights(netD)
    for m in netD.modules():
        if isinstance(m, gn.HipGroupNorm) and m.affine:
            torch.nn.init.normal_(m.weight, 1, 0.2)
            torch.nn.init.normal_(m.bias, 0, 0.2)
    return netD.to(g)


def _plain_copy(netD):
    """The same network in float64 on the CPU from PyTorch's own layers."""
    mods = []
    for m in netD.modules():
        if isinstance(m, dconv.HipConv2d):
            c = torch.nn.Conv2d(m.in_channels, m.out_channels, m.kernel_size, m.stride, m.padding)
            c.load_state_dict(m.state_dict())
            mods.append(c)
        elif isinstance(m, gn.HipGroupNorm):
            c = torch.nn.GroupNorm(m.num_groups, m.num_channels, m.eps, m.affine)
            c.load_state_dict(m.state_dict())
            mods.append(c)
        elif isinstance(m, torch.nn.LeakyReLU):
            mods.append(torch.nn.LeakyReLU(m.negative_slope))
    return torch.nn.Sequential(*mods).double()


def _critic_step(net, real, fake, rp, dtype, device):
    real, fake = real.to(device, dtype), fake.to(device, dtype)
    interp = (rp.to(device, dtype) * fake + (1 - rp.to(device, dtype)) * real).requires_grad_()
    gp = GradientPenaltyLoss(device)(interp, net(interp))
    loss = net(fake).mean() - net(real).mean() + 10 * gp
    return [loss] + list(torch.autograd.grad(loss, list(net.parameters())))


@pytest.mark.parametrize('norm', ['group', 'instance'])
def test_discriminator_step(gpu_device, norm):
    """A WGAN-GP step of the discriminator with a per-sample norm, every gradient against the float64 network, relative
    to its norm and within five times what PyTorch's own float32 network is off (as the batch-norm discriminator's test:
    kinks within float32 rounding of 0 take either slope)."""
    netD = _disc(gpu_device, norm, None)
    g = torch.Generator().manual_seed(5)
    real, fake = torch.rand(3, 3, 80, 72, generator=g), torch.rand(3, 3, 80, 72, generator=g)
    rp = torch.rand(3, 1, 1, 1, generator=g)
    cpu = _plain_copy(netD.cpu())
    netD.to(gpu_device)
    want = _critic_step(cpu, real, fake, rp, torch.float64, 'cpu')
    base = _critic_step(cpu.float(), real, fake, rp, torch.float32, 'cpu')
    got = _critic_step(netD, real, fake, rp, torch.float32, gpu_device)
    rel = lambda a, b: float((a.double().cpu() - b).norm() / b.norm().clamp(min=1e-12))  # noqa: E731
    scale = None
    for (name, _), a, b, f in zip([('loss', 0)] + list(netD.named_parameters()), got, want, base):
        if 'weight' in name:
            scale = float(b.norm())
        if norm == 'instance' and 'bias' in name and float(b.norm()) < 1e-9 * scale:
            # A bias in front of a norm of its own channel has no gradient: what is left are the roundings of its P
            # terms, each at most 8·2^-24 of T (gn_ref), T a few times the gradient reaching the convolution.  The layer's
            # weight gradient sums the same terms times inputs of order 1 over Ci·k² >= 576 taps, so its norm is about
            # sqrt(P·576) terms and the ratio at most 8·2^-24·P·T / (sqrt(P·576)·T/4) = 2e-6·sqrt(P)/24·4 < 1e-4 for
            # P <= 3·40·36 pixels, the floor of every other gradient here.
            assert float(a.norm()) < 1e-4 * scale, (name, float(a.norm()), scale)
            continue
        assert rel(a, b) <= max(1e-4, 5 * rel(f, b)), (name, rel(a, b), rel(f, b))


@pytest.mark.parametrize('norm', ['batch', 'group', 'instance'])
def test_discriminator_with_checkpoints(gpu_device, norm):
    """act_checkpoint changes no forward value, runs the whole WGAN-GP step, repeats bit for bit, and the graph of a
    forward holds less than half of what it did."""
    nets = [_disc(gpu_device, norm, ck) for ck in (None, 'int8')]
    x = torch.rand(4, 3, 96, 96, device=gpu_device)
    held, preds = [], []
    for net in nets:
        net(x)
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        pred = net(x)
        held.append(torch.cuda.memory_allocated() - base)
        preds.append(pred.detach())
        del pred
    assert torch.equal(*preds)
    assert held[1] < (0.75 if norm == 'batch' else 0.5) * held[0], held  # batch norm keeps its fp32 input
    real, fake, rp = x[:2], x[2:], torch.rand(2, 1, 1, 1, device=gpu_device)
    for net in nets:
        net.eval() if norm == 'batch' else net.train()
    a, b = (_critic_step(nets[1], real, fake, rp, torch.float32, gpu_device) for _ in range(2))
    for p, q in zip(a, b):
        assert bool(p.isfinite().all()) and torch.equal(p, q)


def test_carrier_adds_nothing_to_a_first_backward(gpu_device):
    """The stand-in for x that a checkpointed layer saves passes no gradient of zeros on (a pass over x-sized memory and
    an addition to the real one)."""
    from torch.profiler import ProfilerActivity, profile
    x = torch.randn(2, 64, 16, 16, device=gpu_device).contiguous(memory_format=torch.channels_last).requires_grad_()
    y = gn.group_norm_lrelu(x, 32, checkpoint='int8')
    gy = torch.randn_like(y)
    torch.autograd.grad(y, x, gy, retain_graph=True)
    with profile(activities=[ProfilerActivity.CPU]) as prof:
        torch.autograd.grad(y, x, gy)
    names = {e.name for e in prof.events()}
    assert not names & {'aten::zeros', 'aten::fill_', 'aten::add', 'aten::add_', 'aten::copy_'}, names


@pytest.mark.parametrize('norm,ck', [('group', None), ('group', 'int8'), ('instance', 'int8'), ('batch', 'int8')])
def test_training_loop_and_checkpoint_files(gpu_device, tmp_path, norm, ck):
    """SRRaGANModel trains the discriminator with these options (both optimisers step, losses finite), writes it and
    reads it back bit for bit."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), 'golden'))
    from train_recipe import TRAIN_CFGS, step_data, train_opt
    from esr_amd.SRRaGAN_model import SRRaGANModel
    cfg = dict(TRAIN_CFGS['adaptive_rel'], D_update_ratio=1, D_valid_steps=1, min_D_prob_ratio_4_G=0.0,
               min_mean_D_correct=-1.0)
    opt = train_opt(cfg)
    opt['network_D'].update(norm_type=norm, act_checkpoint=ck)
    torch.manual_seed(3)
    model = SRRaGANModel(opt, accumulation_steps_per_batch=1, device=gpu_device)
    before = {k: v.detach().clone() for k, v in model.netD.named_parameters()}
    for k in range(3):
        lr, hr, z = (torch.from_numpy(a).to(gpu_device) for a in step_data(cfg, k))
        model.feed_data({'LR': lr, 'HR': hr, 'Z': z})
        model.optimize_parameters()
    for key in ('l_d_gp', 'l_d_real_fake', 'D_real'):
        if key in model.log_dict:
            assert np.isfinite(np.asarray(model.log_dict[key], dtype=np.float64)).all(), key
    moved = [k for k, v in model.netD.named_parameters() if not torch.equal(v, before[k])]
    weights = [k for k in before if k.endswith('weight')]
    assert set(weights) <= set(moved)
    path = model.save_network(str(tmp_path), model.netD, 'D', 1, model.optimizer_D)
    state = {k: v.detach().clone() for k, v in model.netD.state_dict().items()}
    with torch.no_grad():
        for p in model.netD.parameters():
            p.zero_()
    model.load_network(path, model.netD, optimizer=model.optimizer_D)
    for k, v in model.netD.state_dict().items():
        assert torch.equal(v, state[k]), k
