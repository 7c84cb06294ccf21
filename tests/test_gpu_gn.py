"""Group norm + LeakyReLU on HIP (esr_amd/gn.py) against the float64 definitions of gn_ref.py: forward, backward and
double backward, with the input in float32 and in 8-bit blocks.  Tolerances: one float32 rounding of a float64 result
for y, the rounding bounds derived in gn_ref for the gradients."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import gn_ref as R  # noqa: E402
from esr_amd import act8, gn  # noqa: E402

pytestmark = pytest.mark.gpu

# (N, C, H, W), groups: one value, one channel, ragged blocks (C not a multiple of 32 or 4), groups that no vector
# width divides, more channels than a workgroup has threads, odd maps, several row splits
SHAPES = [((1, 1, 1, 1), 1), ((1, 4, 1, 1), 2), ((2, 3, 5, 7), 3), ((3, 100, 9, 7), 4), ((2, 64, 13, 11), 32),
          ((1, 512, 3, 5), 32), ((2, 37, 6, 5), 1), ((5, 256, 4, 4), 256), ((1, 1025, 2, 3), 25), ((1, 1300, 3, 2), 13),
          ((2, 96, 33, 3), 32), ((1, 64, 70, 65), 8), ((4, 128, 20, 18), 1), ((2, 33, 17, 2), 11), ((33, 8, 2, 2), 4),
          # chunks of lcm(channels of a group, 32) channels; a sample too large for one workgroup and just not
          ((2, 288, 5, 6), 96), ((1, 320, 4, 7), 20), ((3, 192, 9, 2), 16), ((1, 32, 64, 64), 4), ((2, 32, 64, 65), 4),
          ((1, 100, 36, 37), 4), ((2, 40, 60, 61), 5)]


def dev(t, g, nchw=True):
    """float64 NumPy -> float32 on the GPU; NCHW arrays with channels-last storage."""
    t = torch.from_numpy(np.asarray(t, dtype=np.float32)).to(g)
    return t.contiguous(memory_format=torch.channels_last) if nchw else t


def num(t):
    return t.detach().double().cpu().numpy()


def within(mine, ref, tol, what):
    mine = num(mine)
    assert mine.shape == ref.shape, what
    over = np.abs(mine - ref) - (tol + R.U * np.abs(ref) + 1e-13 * np.abs(ref).max(initial=0))
    assert (over <= 0).all(), '%s: %.3g over its bound at %s' % (what, over.max(), np.unravel_index(over.argmax(), over.shape))


def at_blocks(c, f):
    """f with the backward at the values that x's 8-bit blocks hold."""
    sh = c.x.shape
    f.at = R.back(R.pack(R.rows(c.x), lambda v: R.rows(f.pre(R.back(v, sh))))[2], sh)
    return f


def leaves(c, g):
    x = dev(c.x, g).requires_grad_()
    w, b = (None if v is None else dev(v, g, False).requires_grad_() for v in (c.w, c.b))
    return x, w, b


def check(c, g, ck):
    f = R.forward(c)
    x, w, b = leaves(c, g)
    y = gn.group_norm_lrelu(x, c.G, w, b, c.eps, c.slope, ck)
    assert y.permute(0, 2, 3, 1).is_contiguous()
    within(y, f.y, 0, 'y')
    if ck:
        at_blocks(c, f)
    d = R.backward(c, f)
    gy = dev(c.gy, g).requires_grad_()
    ps = [t for t in (w, b) if t is not None]
    gx, *gp = torch.autograd.grad(y, [x] + ps, gy, create_graph=True)
    within(gx, d.gx, d.tol_gx, 'gx')
    if ps:
        within(gp[0], d.gw, d.tol_gw, 'dgamma')
        within(gp[1], d.gb, d.tol_gb, 'dbeta')
    for use in ((True, True, True), (True, False, False), (False, True, True)):
        if not ps and not use[0]:
            continue
        L = (gx * dev(c.u, g)).sum() if use[0] else 0
        use = (use[0], use[1] and bool(ps), use[2] and bool(ps))
        if use[1]:
            L = L + (gp[0] * dev(c.ga, g, False)).sum() + (gp[1] * dev(c.gb, g, False)).sum()
        e = R.backward2(c, f, d, *use)
        got = torch.autograd.grad(L, [x, gy] + ([w] if ps else []), retain_graph=True)
        within(got[0], e.g_x, e.tol_x, 'g_x %s' % (use,))
        within(got[1], e.g_gy, e.tol_gy, 'g_gy %s' % (use,))
        if ps:
            within(got[2], e.g_w, e.tol_w, 'g_gamma %s' % (use,))


@pytest.mark.parametrize('ck', [None, 'int8'])
@pytest.mark.parametrize('shape,G', SHAPES)
def test_against_definition(gpu_device, shape, G, ck):
    check(R.case(shape, G, seed=sum(shape), dtype=np.float32), gpu_device, ck)


@pytest.mark.parametrize('ck', [None, 'int8'])
@pytest.mark.parametrize('kw', [{'affine': False}, {'slope': 0.0}, {'slope': 1.0}, {'slope': 1.5}, {'eps': 1e-2},
                                {'scale': 1e-3, 'shift': 30.0}, {'scale': 1e-6}, {'scale': 1e12}])
def test_parameters_and_ranges(gpu_device, kw, ck):
    check(R.case((2, 40, 7, 5), 8, seed=5, dtype=np.float32, **kw), gpu_device, ck)


@pytest.mark.parametrize('ck', [None, 'int8'])
def test_constant_groups_and_zero_kinks(gpu_device, ck):
    """A constant group normalises to β; a pre-activation of exactly 0 takes the slope, as LeakyReLU's gradient does."""
    c = R.case((2, 8, 4, 4), 4, seed=1, dtype=np.float32)
    c.x[0, :2] = 3.25
    c.x[1, 2:4] = np.tile([-1.0, 0.0, 1.0, 0.0], 8).reshape(2, 4, 4)
    c.b[2:4] = 0.0
    check(c, gpu_device, ck)


@pytest.mark.parametrize('ck', [None, 'int8'])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_nonfinite_stays_in_its_group(gpu_device, bad, ck):
    c = R.case((2, 64, 5, 3), 4, seed=2, dtype=np.float32)
    x, w, b = leaves(c, gpu_device)
    y0 = gn.group_norm_lrelu(x, 4, w, b, c.eps, c.slope, ck)
    gx0, = torch.autograd.grad(y0, x, dev(c.gy, gpu_device))
    with torch.no_grad():
        x[1, 20, 2, 1] = bad
    y = gn.group_norm_lrelu(x, 4, w, b, c.eps, c.slope, ck)
    gx, = torch.autograd.grad(y, x, dev(c.gy, gpu_device))
    hit = torch.zeros_like(x, dtype=torch.bool)
    hit[1, 16:32] = True
    assert torch.equal(y[~hit], y0[~hit]) and bool(y[hit].isnan().all())
    if ck:  # the block that holds it reads back as NaN: the groups of 16 channels share blocks of 32
        other = hit.clone()
        other[1, :16, 2, 1] = True
        assert torch.equal(gx[~other][~gx[~other].isnan()], gx0[~other][~gx[~other].isnan()])
        assert bool(gx[0].eq(gx0[0]).all()) and bool(gx[1, 32:].eq(gx0[1, 32:]).all())
    else:
        assert torch.equal(gx[~hit], gx0[~hit])
    assert bool(gx[hit].isnan().all())


@pytest.mark.parametrize('shape,G', SHAPES)
def test_output_blocks(gpu_device, shape, G):
    """out8: y's blocks from the norm's pass are act8.pack's of y, y itself unchanged."""
    c = R.case(shape, G, seed=7, dtype=np.float32)
    x, w, b = leaves(c, gpu_device)
    for ck in (None, 'int8'):
        y, y8 = gn.group_norm_lrelu(x, G, w, b, c.eps, c.slope, ck, out8=True)
        want = act8.pack(y.permute(0, 2, 3, 1))
        assert torch.equal(y8.codes, want.codes) and torch.equal(y8.exps, want.exps)
        plain = gn.group_norm_lrelu(x, G, w, b, c.eps, c.slope, ck)
        assert torch.equal(y, plain)
        gy = dev(c.gy, gpu_device)
        assert torch.equal(torch.autograd.grad(y, x, gy)[0], torch.autograd.grad(plain, x, gy)[0])


@pytest.mark.parametrize('ck', [None, 'int8'])
def test_masks_of_blocks_are_the_forwards(gpu_device, ck):
    """The slope of every value is the forward's, bit for bit: with one group per channel, γ = 1 and M large, gy picks
    out single values' slopes through dβ."""
    c = R.case((1, 64, 40, 40), 64, seed=8, dtype=np.float32, shift=0.0)
    c.w[:], c.b[:] = 1.0, 0.01
    x, w, b = leaves(c, gpu_device)
    y = gn.group_norm_lrelu(x, 64, w, b, c.eps, c.slope, ck)
    z = y.detach() > 0
    sel = torch.rand(6, *x.shape, device=gpu_device) < 0.01
    for s in sel:
        gb, = torch.autograd.grad(y, b, s.float(), retain_graph=True)
        want = torch.where(z, 1.0, float(np.float32(c.slope))).double() * s
        assert torch.equal(gb, want.sum((0, 2, 3)).float())


def test_blocks_next_to_the_largest_float(gpu_device):
    """The kink between the largest code's value, 63/64 · 2^128, and the largest float: no code on the float's side of it
    is finite, so the largest one stays (x̂ = 0.97 of ±1 with β = −0.98), and the gradients stay finite."""
    top = float(np.finfo(np.float32).max)
    for W in (2, 4096):  # one launch, three launches
        x = torch.zeros(1, 32, 64, W, device=gpu_device).contiguous(memory_format=torch.channels_last)
        x[..., W // 2:] = top
        x.requires_grad_()
        w = torch.ones(32, device=gpu_device, requires_grad=True)
        b = torch.full((32,), -0.98, device=gpu_device, requires_grad=True)
        y, y8 = gn.group_norm_lrelu(x, 32, w, b, 1e-5, 0.25, 'int8', out8=True)
        assert torch.isfinite(y).all() and torch.isfinite(y8.unpack()).all()
        # x̂ is −1 and 0.96875 at the codes' values, both on the slope's side
        _, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
        half = 64 * W // 2
        assert torch.equal(gb, torch.full_like(gb, 0.25 * 2 * half))
        assert torch.allclose(gw, torch.full_like(gw, 0.25 * half * -0.03125), rtol=1e-5, atol=0)


def test_layouts_and_offsets(gpu_device):
    """NCHW storage, channel slices, transposed maps and bases off 16 bytes give the channels-last result bit for bit."""
    c = R.case((2, 24, 6, 5), 4, seed=4, dtype=np.float32)
    x, w, b = leaves(c, gpu_device)
    x = x.detach()
    wide = torch.randn(2, 40, 6, 5, device=gpu_device)
    wide[:, 9:33] = x
    flat = torch.empty(x.numel() + 1, device=gpu_device)[1:]
    off = flat.view(2, 6, 5, 24).copy_(x.permute(0, 2, 3, 1)).permute(0, 3, 1, 2)
    wt = x.transpose(2, 3).contiguous().transpose(2, 3)
    gy = dev(c.gy, gpu_device)
    outs = []
    for ck in (None, 'int8'):
        for v in (x, x.contiguous(), wide[:, 9:33], wide.contiguous(memory_format=torch.channels_last)[:, 9:33], off, wt):
            v = v.detach().requires_grad_()
            for g in (gy, gy.contiguous()):
                y = gn.group_norm_lrelu(v, 4, w, b, c.eps, c.slope, ck)
                outs.append((ck, y, *torch.autograd.grad(y, (v, w, b), g)))
    for a in outs:
        first = outs[0] if a[0] is None else outs[12]
        for p, q in zip(a[1:], first[1:]):
            assert torch.equal(p, q)


def test_empty_batch_and_no_grad(gpu_device):
    x = torch.empty(0, 8, 4, 4, device=gpu_device, requires_grad=True)
    y = gn.group_norm_lrelu(x, 4, checkpoint='int8')
    assert y.shape == x.shape
    y.sum().backward()
    assert x.grad.shape == x.shape
    c = R.case((2, 8, 4, 4), 4, dtype=np.float32)
    xs, w, b = leaves(c, gpu_device)
    with torch.no_grad():
        y = gn.group_norm_lrelu(xs, 4, w, b, c.eps, c.slope, 'int8')
    assert not y.requires_grad
    within(y, R.forward(c).y, 0, 'y')
    layer = gn.HipGroupNorm(4, 8).to(gpu_device)
    ref = torch.nn.GroupNorm(4, 8).double()
    torch.testing.assert_close(layer(xs).detach().cpu().double(), ref(torch.from_numpy(c.x)), rtol=2 ** -22, atol=1e-6)


def test_checkpoint_frees_the_input(gpu_device):
    """With a checkpoint the graph holds 33/32 bytes per value of x, not 4."""
    x = torch.randn(4, 64, 128, 128, device=gpu_device).contiguous(memory_format=torch.channels_last)
    held = {}
    for ck in (None, 'int8'):
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        src = (x * 2.0).requires_grad_()
        y = gn.group_norm_lrelu(src * 1.0, 32, checkpoint=ck)  # the product's storage lives on only if it is saved
        held[ck] = torch.cuda.memory_allocated() - base - 2 * x.numel() * 4
        del y, src
    assert held[None] >= 4 * x.numel()
    assert held['int8'] <= 1.1 * x.numel() * 33 / 32


def test_deterministic_and_streams(gpu_device):
    """Repeated and concurrent calls on two streams give the first call's bits."""
    c = R.case((4, 128, 60, 61), 32, seed=11, dtype=np.float32)
    x, w, b = leaves(c, gpu_device)
    gy = dev(c.gy, gpu_device)

    def run(ck):
        y = gn.group_norm_lrelu(x, 32, w, b, c.eps, c.slope, ck)
        return (y,) + torch.autograd.grad(y, (x, w, b), gy)
    want = {ck: run(ck) for ck in (None, 'int8')}
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s, ck in zip(streams, (None, 'int8')):
            with torch.cuda.stream(s):
                got.append((ck, run(ck)))
    torch.cuda.synchronize()
    for ck, o in got:
        for p, q in zip(o, want[ck]):
            assert torch.equal(p, q)


@pytest.mark.parametrize('ck', [None, 'int8'])
def test_graph_capture(gpu_device, ck):
    """Forward, backward and double backward captured once and replayed between eager calls on new inputs."""
    c = R.case((2, 64, 24, 20), 32, seed=6, dtype=np.float32)
    x0, w0, b0 = (t.detach() for t in leaves(c, gpu_device))
    static = [x0.clone(memory_format=torch.preserve_format), dev(c.gy, gpu_device), dev(c.u, gpu_device)]

    def step(x, gy, u):
        x, gy = x.detach().requires_grad_(), gy.detach().requires_grad_()
        w, b = w0.detach().requires_grad_(), b0.detach().requires_grad_()
        y = gn.group_norm_lrelu(x, 32, w, b, c.eps, c.slope, ck)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
        return (y.detach(), gx.detach(), gw.detach(), gb.detach()) + torch.autograd.grad(gx, (x, gy, w), u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for k in range(4):
        new = [torch.randn_like(t) * (k + 1) for t in static]
        want = step(*new)
        for s, n in zip(static, new):
            s.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, want):
            assert torch.equal(p, q)


def test_difference_quotient(gpu_device):
    """The GPU's gradient against central differences of the float64 forward."""
    c = R.case((2, 32, 6, 6), 8, seed=21, dtype=np.float32)
    x, w, b = leaves(c, gpu_device)
    y = gn.group_norm_lrelu(x, 8, w, b, c.eps, c.slope)
    grads = torch.autograd.grad(y, (x, w, b), dev(c.gy, gpu_device))
    rng = np.random.default_rng(2)
    for name, g in zip('xwb', grads):
        v, base, t, loss = rng.standard_normal(tuple(g.shape)), getattr(c, name), 1e-6, []
        for s in (t, -t):
            setattr(c, name, base + s * v)
            loss.append((R.forward(c).y * c.gy).sum())
        setattr(c, name, base)
        # float32 rounding of every gradient value (8 roundings of terms a few times its size) on top of the quotient's
        np.testing.assert_allclose((loss[0] - loss[1]) / (2 * t), (num(g) * v).sum(),
                                   atol=1e-6 * np.abs(num(g) * v).sum() + 1e-6)


def test_refuses_other_types_and_third_order(gpu_device):
    x = torch.randn(2, 8, 4, 4, device=gpu_device)
    for bad in (x.half(), x.double(), x.bfloat16()):
        with pytest.raises(RuntimeError, match='float32'):
            gn.group_norm_lrelu(bad, 4)
    with pytest.raises(RuntimeError, match='float32'):
        gn.group_norm_lrelu(x, 4, torch.ones(8))
    x.requires_grad_()
    gx, = torch.autograd.grad(gn.group_norm_lrelu(x, 4).pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match='twice'):
        torch.autograd.grad(gx.pow(2).sum(), x, create_graph=True)
