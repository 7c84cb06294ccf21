"""How the discriminator walks its layers (discriminator._run): which calls the modules get, and that hooks fire as in
nn.Sequential.  The layers' kernels are replaced by plain functions, so the walk runs on the CPU."""
import torch
import torch.nn as nn

from esr_amd import act8, discriminator
from esr_amd.dconv import HipConv2d
from esr_amd.gn import HipGroupNorm


class Conv(HipConv2d):
    """Records what it is called with; adds 1."""

    def forward(self, x, x8=None):
        self.got = (x, x8)
        return x + 1


class PlainConv(HipConv2d):
    """A subclass whose forward takes the input alone."""

    def forward(self, x):
        self.got = x
        return x + 1


class Norm(HipGroupNorm):
    """2x in place of the norm; its blocks are the output they belong to."""

    def lrelu(self, x, slope, out8=False):
        y = torch.where(x > 0, 2 * x, 2 * slope * x)
        return (y, ('blocks of', y)) if out8 else y


def net(conv=Conv, ck='int8'):
    mods = [conv(4, 4, 3, padding=1), Norm(2, 4, checkpoint=ck), nn.LeakyReLU(0.5, True), conv(4, 4, 3, padding=1)]
    for m in mods:
        if isinstance(m, HipConv2d):
            m.act_checkpoint = ck
    return nn.Sequential(*mods)


X = torch.tensor([-3.0, 2.0, 5.0, -1.0]).view(1, 4, 1, 1)
WANT = torch.tensor([-2.0, 6.0, 12.0, 0.0]).view(1, 4, 1, 1)  # what reaches the second convolution


def test_blocks_go_to_the_convolution_behind_the_norm():
    seq = net()
    discriminator._run(seq, X)
    assert torch.equal(seq[3].got[0], WANT) and seq[3].got[1][1] is seq[3].got[0] and seq[0].got[1] is None


def test_convolutions_without_blocks_get_the_input_alone():
    for ck in (None, 'int8'):
        seq = net(PlainConv, ck)
        if ck:
            seq[3].weight.requires_grad_(False)  # keeps nothing
        discriminator._run(seq, X)
        assert torch.equal(seq[3].got, WANT)
    seq = net(ck=None)
    seen = []
    seq[3].register_forward_pre_hook(lambda m, args: seen.append(args))
    discriminator._run(seq, X)
    assert [len(a) for a in seen] == [1]


def test_a_hook_that_changes_the_input_leaves_no_blocks_of_the_old_one():
    seq = net()
    seq[3].register_forward_pre_hook(lambda m, args: (args[0] * 3,))
    discriminator._run(seq, X)
    assert torch.equal(seq[3].got[0], 3 * WANT) and seq[3].got[1] is None
    # in place: the blocks that the norm's pass would have written are those of the values before
    seq = net()
    seq[3].register_forward_pre_hook(lambda m, args: (args[0].mul_(3),))
    discriminator._run(seq, X)
    assert torch.equal(seq[3].got[0], 3 * WANT) and seq[3].got[1] is None
    # a hook for all modules
    h = nn.modules.module.register_module_forward_pre_hook(
        lambda m, args: (args[0] * 3,) if isinstance(m, Conv) else None)
    try:
        seq = net()
        discriminator._run(seq, X)
    finally:
        h.remove()
    assert seq[3].got[1] is None


def test_hooks_of_the_norm_and_its_activation_fire():
    want = discriminator._run(net(), X)
    for at in (1, 2):
        for kind in ('register_forward_hook', 'register_forward_pre_hook'):
            seq, seen = net(), []
            getattr(seq[at], kind)(lambda m, *args: seen.append(m))
            assert torch.equal(discriminator._run(seq, X), want) and seen == [seq[at]]
    seq = net()
    seq[1].register_forward_hook(lambda m, args, y: -y)  # a hook that changes the norm's result
    out = discriminator._run(seq, X)
    plain = nn.functional.leaky_relu(-2 * (X + 1), 0.5) + 1
    assert torch.equal(out, plain) and seq[3].got[1] is None
    seq, seen = net(), []
    x = X.clone().requires_grad_()
    seq[1].register_full_backward_hook(lambda m, gi, go: seen.append(m))
    discriminator._run(seq, x).sum().backward()
    assert seen == [seq[1]]


def test_a_group_of_one_value_is_refused():
    """128 x 128 crops through four strides leave the classifier's 8x8 layer a 1 x 1 map: an instance norm there makes
    the score the same for every input and its gradient 0."""
    import pytest

    from esr_amd.discriminator import Discriminator_VGG_128_
    for layer, x in ((HipGroupNorm(4, 4), torch.zeros(2, 4, 1, 1)), (HipGroupNorm(1, 1), torch.zeros(2, 1, 1, 1)),
                     (HipGroupNorm(4, 4, affine=False).eval(), torch.zeros(2, 4, 1, 1))):
        for call in (layer, lambda t, layer=layer: layer.lrelu(t, 0.2)):
            with pytest.raises(ValueError, match='one value'):
                call(x)
    # the discriminator: shapes alone, the convolutions' of PyTorch and the norms' check
    for norm, groups, refused in (('instance', 32, True), ('group', 32, False), ('group', 100, True)):
        netD = Discriminator_VGG_128_(3, 64, norm_type=norm, nb=8, num_2_strides=4, norm_groups=groups)

        def walk(seq, x):
            for m in seq.children():
                if isinstance(m, nn.Sequential):
                    x = walk(m, x)
                elif isinstance(m, HipConv2d):
                    x = torch.empty(x.shape[0], m.out_channels, *((n + 2 * m.padding[0] - m.kernel_size[0]) //
                                                                  m.stride[0] + 1 for n in x.shape[2:]))
                elif isinstance(m, HipGroupNorm):
                    m.check(x)
            return x

        def score():
            return walk(netD.classifier, walk(netD.features, torch.empty(2, 3, 128, 128))).shape
        if refused:
            with pytest.raises(ValueError, match='one value'):
                score()
        else:
            assert score() == (2, 1, 1, 1)


def test_layers_saved_whole_before_they_had_checkpoints():
    """A pickled discriminator's convolutions without the attribute keep fp32."""
    m = HipConv2d(4, 4, 3, padding=1)
    m.__dict__.pop('act_checkpoint', None)
    assert m.act_checkpoint is None and not m.keeps8()


def test_empty_batch_has_gradients_of_zero(monkeypatch):
    """No images: the norm's weight and bias get gradients of zero, as nn.GroupNorm's do, not none."""
    from esr_amd import gn
    monkeypatch.setattr(act8, 'check_dev', lambda what, *ts: ts[0].device)
    for out8 in (False, True):
        x = torch.zeros(0, 4, 3, 2, requires_grad=True)
        w, b = torch.ones(4, requires_grad=True), torch.zeros(4, requires_grad=True)
        y = gn.group_norm_lrelu(x, 2, w, b, out8=out8)
        y = y[0] if out8 else y
        assert y.shape == x.shape
        gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
        assert gx.shape == x.shape and torch.equal(gw, torch.zeros(4)) and torch.equal(gb, torch.zeros(4))
    assert gn.group_norm_lrelu(x, 2).shape == x.shape
