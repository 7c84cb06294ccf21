"""The discriminator with 8-bit checkpoints from PyTorch's operations on the CPU, in float64 or float32: what a layer keeps
in 8 bits is read at its blocks' values (gn_ref.pack) by the backward and the double backward, whose derivatives go on to
the values themselves."""
import os
import sys

import torch
import torch.nn as nn

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import gn_ref as R  # noqa: E402
from esr_amd import dconv, gn  # noqa: E402


def at_blocks(x, pre=None):
    """x with the values of its 8-bit blocks (NCHW, blocks along the channels; pre: what keeps its sign) and with the
    derivative of x."""
    shape = tuple(x.shape)
    side = None if pre is None else (lambda v: R.rows(pre(torch.from_numpy(R.back(v, shape)).to(x.dtype)).numpy()))
    q = torch.from_numpy(R.back(R.pack(R.rows(x.detach().numpy()), side)[2], shape)).to(x.dtype)
    return x + (q - x).detach()


class Conv(nn.Conv2d):
    keep = None  # 'int8': the weight gradient is that of the input's blocks

    def forward(self, x):
        y = super().forward(x)
        if self.keep is None:
            return y
        y8 = super().forward(self.kept(x))
        return y8 + (y - y8).detach()

    def kept(self, x):
        return at_blocks(x)


class _Norm8(torch.autograd.Function):
    """lrelu(gn(x)) whose backward is that at xq, with x's statistics, which have in the double backward the derivatives of a
    mean and of a deviation."""

    @staticmethod
    def forward(ctx, x, xq, w, b, mu, r, G, slope):
        z = (x - mu) * r * w + b
        ctx.save_for_backward(xq, w, mu, r, z > 0)
        ctx.G, ctx.slope = G, slope
        return torch.where(z > 0, z, slope * z)

    @staticmethod
    def backward(ctx, gy):
        xq, w, mu, r, up = ctx.saved_tensors
        mean = lambda t: _group(t, ctx.G)  # noqa: E731
        d = xq - xq.detach()
        r_at = 1 / (1 / r + mean(d * (xq.detach() - mu) * r))
        xh = (xq - mu - mean(d)) * r_at
        gz = torch.where(up, gy, ctx.slope * gy)
        h = gz * w
        gx = r_at * (h - mean(h) - xh * mean(h * xh))
        ch = lambda t: t.sum((0, 2, 3), keepdim=True)  # noqa: E731
        return gx, None, ch(gz * xh), ch(gz), None, None, None, None


def _group(t, G):
    """The mean over each (sample, group), for every value."""
    n, c = t.shape[:2]
    return t.reshape(n, G, -1).mean(2).repeat_interleave(c // G, 1)[:, :, None, None]


class Norm(nn.GroupNorm):
    """GroupNorm and the LeakyReLU behind it, the input kept in 8 bits."""
    slope = 0.2

    def forward(self, x):
        G, v = self.num_groups, x.detach()
        mu = _group(v, G)
        r = 1 / torch.sqrt(_group((v - mu) ** 2, G) + self.eps)
        w, b = ((torch.full((1,), one, dtype=x.dtype) if t is None else t).view(1, -1, 1, 1)
                for t, one in ((self.weight, 1.0), (self.bias, 0.0)))
        return _Norm8.apply(x, self.kept(x, lambda t: (t - mu) * r * w.detach() + b.detach()), w, b, mu, r, G, self.slope)

    def kept(self, x, pre):
        return at_blocks(x, pre)


def network(netD, conv=Conv, norm=Norm):
    """netD's layers with its parameters, in float64 on the CPU; convolutions and group norms keep what netD's keep."""
    mods, fused = [], False
    for m in netD.modules():
        if isinstance(m, dconv.HipConv2d):
            c = conv(m.in_channels, m.out_channels, m.kernel_size, m.stride, m.padding)
            # (the first block's mask is exact in 8 bits, and its input is not kept so)
            c.keep = None if dconv.dfirst_ok(m) else m.act_checkpoint
        elif isinstance(m, gn.HipGroupNorm):
            c = (norm if m.checkpoint else nn.GroupNorm)(m.num_groups, m.num_channels, m.eps, m.affine)
        elif isinstance(m, nn.BatchNorm2d):
            c = nn.BatchNorm2d(m.num_features, m.eps)
        elif isinstance(m, nn.LeakyReLU):
            if fused:  # in the norm
                fused = False
                continue
            c = nn.LeakyReLU(m.negative_slope)
        else:
            continue
        c.load_state_dict({k: v.cpu() for k, v in m.state_dict().items()})
        fused = isinstance(c, Norm)
        mods.append(c)
    return nn.Sequential(*mods).double()
