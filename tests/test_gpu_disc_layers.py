"""The discriminator's layers as they are put together: upstream gradients of every layout, hooks, derivatives of every
order, 8-bit checkpoints against the definitions of gn_ref.py."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import disc_ref  # noqa: E402
import test_disc_ref_host as T  # noqa: E402
from esr_amd import act8, bn, dconv, gn  # noqa: E402

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


@pytest.mark.parametrize('k,s,p', [(3, 1, 1), (4, 2, 1)])
def test_conv_checkpoint_third_order(gpu_device, k, s, p):
    """A convolution that keeps its input in 8 bits, on values that the blocks hold exactly: every term of its third
    derivatives is there (the plain layer's, up to what two evaluations of its products differ by)."""
    torch.manual_seed(k)
    m = dconv.HipConv2d(64, 32, k, stride=s, padding=p).to(gpu_device)
    x0 = act8.pack(torch.randn(2, 10, 12, 64, device=gpu_device)).unpack().permute(0, 3, 1, 2)
    gy0 = torch.randn_like(m(x0))
    ups = [torch.randn_like(t) for t in (x0, m.weight, m.bias)]
    ups2 = [torch.randn_like(t) for t in (x0, m.weight, gy0)]
    res = []
    for ck in (None, 'int8'):
        m.act_checkpoint = ck
        x, gy = x0.detach().requires_grad_(), gy0.detach().requires_grad_()
        u = [t.detach().requires_grad_() for t in ups]
        first = torch.autograd.grad(m(x), (x, m.weight, m.bias), gy, create_graph=True)
        second = torch.autograd.grad(sum((a * b).sum() for a, b in zip(first, u)), (x, m.weight, gy), create_graph=True)
        res.append(first + second + torch.autograd.grad(sum((a * b).sum() for a, b in zip(second, ups2)),
                                                        [x, m.weight, gy] + u))
    for i, (a, b) in enumerate(zip(*res)):
        # both split each operand into f16 pieces that keep 2^-21 of it or better; the sums have at most 2·10·12 = 240 or
        # 64·k² = 1024 terms, each rounded by 2^-24 of a partial sum: sqrt(1024) of them in the mean; a third derivative
        # goes through up to two such products, and both evaluations err: 4
        a, b = a.detach(), b.detach()
        assert float((a - b).norm()) <= (2 * 2.0 ** -21 + 32 * 2.0 ** -24) * 4 * float(b.norm()) + 1e-12, i


def test_score_depends_on_the_input_or_is_refused(gpu_device):
    """128 x 128 crops through four strides: the head's map is 1 x 1.  Group norm's critic answers to its input there;
    instance norm's could not, and is refused."""
    from esr_amd.discriminator import Discriminator_VGG_128_
    torch.manual_seed(1)
    x = torch.rand(2, 3, 128, 128, device=gpu_device).requires_grad_()
    mk = lambda norm: Discriminator_VGG_128_(3, 64, norm_type=norm, nb=8, num_2_strides=4).to(gpu_device)  # noqa: E731
    y = mk('group')(x)
    gx, = torch.autograd.grad(y.sum(), x)
    y = y.detach()
    assert y.shape == (2, 1, 1, 1) and float(y[0]) != float(y[1]) and float(gx[0].norm()) > 0 and float(gx[1].norm()) > 0
    with pytest.raises(ValueError, match='one value'):
        mk('instance')(x)


def test_checkpoint_holds_blocks_and_statistics(gpu_device):
    """What a forward with a checkpoint leaves allocated beside its input and output, in the bytes that were asked for (the
    allocator may hand out larger blocks that it has cached: one is left for it here)."""
    requested = lambda: torch.cuda.memory_stats()['requested_bytes.all.current']  # noqa: E731
    x = cl(torch.randn(4, 64, 128, 128, device=gpu_device))
    codes, exps = x.numel(), x.numel() // 32
    gn.group_norm_lrelu(x, 32)
    src = (x * 2.0).requires_grad_()
    for ck, kept in ((None, 4 * x.numel()), ('int8', codes + exps + 4)):
        spare = torch.empty(codes + (7 << 17), dtype=torch.uint8, device=gpu_device)
        base = requested()
        del spare
        y = gn.group_norm_lrelu(src * 1.0, 32, checkpoint=ck)  # the product's storage lives on only if it is saved
        held = requested() - base + codes + (7 << 17) - 4 * x.numel()
        assert held == kept + 2 * 4 * 32 * 8, (ck, held)  # μ and r of every (sample, group), float64
        del y


@pytest.mark.parametrize('norm', ['batch', 'group', 'instance'])
def test_discriminator_with_checkpoints_against_its_definition(gpu_device, norm):
    """A WGAN-GP step of the discriminator that keeps its activations in 8 bits: every gradient is the float64 network's that
    reads the blocks' values in its backward and double backward (the host test of that network says what would show)."""
    netD = T.discriminator(norm, 'int8')
    want = T.step(disc_ref.network(netD))
    got = [t.detach() for t in T.critic_step(netD.to(gpu_device), *T.data(), torch.float32, gpu_device)]
    assert [tuple(t.shape) for t in got] == [tuple(t.shape) for t in want]
    far = T.apart(got, want, norm)
    assert far <= T.BOUND[norm], far


@pytest.mark.parametrize('bad', [None, float('nan'), float('inf')])
def test_first_block_checkpoint_is_exact(gpu_device, bad):
    """The first block keeps its output's sign in 8 bits: output, gradients and double backward bit for bit those of the
    block that keeps its output."""
    torch.manual_seed(2)
    conv = dconv.HipConv2d(3, 64, 3, padding=1).to(gpu_device)
    x0 = cl(torch.rand(2, 3, 21, 18, device=gpu_device))
    if bad is not None:
        x0[1, 2, 5, 7] = bad
    gy0 = cl(torch.randn(2, 64, 21, 18, device=gpu_device))
    ups = [torch.randn_like(t) for t in (x0, conv.weight, conv.bias)]
    res = []
    for ck in (None, 'int8'):
        conv.act_checkpoint = ck
        x, gy = x0.detach().requires_grad_(), gy0.detach().requires_grad_()
        y, y8 = dconv.dfirst_lrelu8(x, conv, 0.2)
        assert (y8 is not None) == bool(ck)
        first = torch.autograd.grad(y, (x, conv.weight, conv.bias), gy, create_graph=True)
        second = torch.autograd.grad(sum((a * b).sum() for a, b in zip(first, ups)), (x, gy, conv.weight))
        res.append([y, *first, *second])
    if ck and bad is None:
        assert torch.equal(y8.codes, act8.pack(y.detach().permute(0, 2, 3, 1)).codes)
    for i, (a, b) in enumerate(zip(*res)):
        a, b = a.detach(), b.detach()
        if bad is None:
            assert torch.equal(a, b), i
        else:  # the whole block of a non-finite value reads back as NaN: at its pixels the slope of the others is lost
            assert torch.equal(a[0], b[0]) or i in (2, 3, 6), i


@pytest.mark.parametrize('prec', ['x6', 'f32'])
def test_conv_checkpoint_in_another_precision(gpu_device, prec):
    """The weight gradient of a layer set to x6 or f32 is that arithmetic's, of the blocks' values."""
    torch.manual_seed(4)
    m = dconv.HipConv2d(64, 32, 3, padding=1).to(gpu_device)
    m.act_checkpoint, m.esr_precision = 'int8', prec
    x = cl(torch.randn(2, 64, 14, 11, device=gpu_device))
    gy = cl(torch.randn(2, 32, 14, 11, device=gpu_device))
    gw, = torch.autograd.grad(m(x), m.weight, gy)
    v = act8.pack(x.permute(0, 2, 3, 1)).unpack()
    assert torch.equal(gw, dconv.conv_wgrad(v, gy.permute(0, 2, 3, 1), 3, 1, 1, prec))


def test_two_threads(gpu_device):
    """Two host threads with the layers on one stream, and on streams of their own: every result is the first call's."""
    import threading
    torch.manual_seed(6)
    x0, gy0 = cl(torch.randn(2, 64, 40, 37, device=gpu_device)), cl(torch.randn(2, 32, 40, 37, device=gpu_device))
    m = dconv.HipConv2d(64, 32, 3, padding=1).to(gpu_device)
    m.act_checkpoint = 'int8'

    def step(ck):
        x = x0.detach().requires_grad_()
        y, y8 = gn.group_norm_lrelu(x, 8, checkpoint=ck, out8=True)
        out = m(y, y8)
        gx, gw = torch.autograd.grad(out, (x, m.weight), gy0, create_graph=True)
        return [t.detach() for t in (out, gx, gw)] + list(torch.autograd.grad(gx.pow(2).sum() + gw.sum(), (x, m.weight)))
    want = {ck: step(ck) for ck in (None, 'int8')}
    torch.cuda.synchronize()
    got, errors = [], []

    def run(ck, stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(12):
                    got.append((ck, step(ck)))
                    torch.empty(1 << 16, device=gpu_device).fill_(float('nan'))  # a neighbour of the workspaces
        except Exception as e:  # noqa: BLE001
            errors.append(e)
    for streams in ([torch.cuda.current_stream()] * 2, [torch.cuda.Stream(), torch.cuda.Stream()]):
        threads = [threading.Thread(target=run, args=a) for a in zip((None, 'int8'), streams)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
    assert not errors and len(got) == 48
    for ck, outs in got:
        for i, (a, b) in enumerate(zip(outs, want[ck])):
            assert torch.equal(a, b), (ck, i)
