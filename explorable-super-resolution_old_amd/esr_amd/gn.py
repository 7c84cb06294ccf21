"""GroupNorm + LeakyReLU of channels-last activations, fused on HIP (csrc/esr_gn.hip): forward, backward and the
backward's own backward, which the WGAN-GP penalty needs (loss.py:244-263).

The norm for a critic under a gradient penalty: the penalty bounds the gradient of each sample's score, and a batch norm
makes that score a function of the other samples.  Statistics are per (sample, group of channels), so a layer has no
running buffers, is the same in training and eval mode, and is the same on every rank.  One group per channel without
affine parameters is instance norm (block.py:46-58).  With checkpoint='int8' the layer keeps its input in 8 bits (act8.py)
instead of fp32 until its backward."""
import functools
import math

import torch
import torch.nn as nn

from . import _lib
from . import act8


def _p(t):
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=256)
def _ws_bytes(N, HW, C, G):
    n = int(_lib.load().esr_gn_workspace_bytes(N, HW, C, G))
    if n < 0:
        raise RuntimeError('esr_gn_workspace_bytes failed with esr_status %d for N, HW, C = %d, %d, %d in %d groups'
                           % (n, N, HW, C, G))
    return n


def _bytes(n, dev):
    return torch.empty(n, device=dev, dtype=torch.uint8)


def _nhwc(t):
    """t NCHW with channels-last storage (a copy of one in another layout)."""
    return t if t.is_contiguous(memory_format=torch.channels_last) else \
        t.contiguous(memory_format=torch.channels_last)


def _bwd(src, codes, exps, gamma, beta, stat, gy, G, slope, keep):
    """(gx, dγ, dβ, sums) of esr_gn_lrelu_bwd; the sums as a tensor of their own if `keep`, for the double backward."""
    N, C, H, W = gy.shape
    dev = gy.device
    n, k = _ws_bytes(N, H * W, C, G), 16 * N * C
    gx = torch.empty_like(gy)
    gg = torch.empty(C, device=dev, dtype=torch.float32)
    gb = torch.empty(C, device=dev, dtype=torch.float32)
    ws = _bytes(n if keep else n + k, dev)
    sums = _bytes(k, dev) if keep else None
    with act8.on(dev):
        _lib.check(_lib.load().esr_gn_lrelu_bwd(_p(src) if codes is None else None, _p(codes), _p(exps), gy.data_ptr(),
                                                N, H * W, C, G, _p(gamma), _p(beta), stat.data_ptr(), slope,
                                                gx.data_ptr(), gg.data_ptr(), gb.data_ptr(),
                                                sums.data_ptr() if keep else ws.data_ptr() + n, ws.data_ptr(),
                                                act8.stream(dev)), 'esr_gn_lrelu_bwd')
    return gx, gg, gb, sums


class _GNLReLUFn(torch.autograd.Function):
    """NCHW (channels-last storage) -> lrelu(gn(x)).  `carrier` is None, or act8.Carrier's stand-in for x: then x is kept
    in 8 bits.  out8: the result is (y, codes, exps) with y's 8-bit blocks [N, H, W, C]."""

    @staticmethod
    def forward(ctx, x, carrier, gamma, beta, G, eps, slope, out8):
        N, C, H, W = x.shape
        dev = x.device
        y = torch.empty_like(x)
        stat = torch.empty(2 * N * G, device=dev, dtype=torch.float64)
        codes, exps = act8.empty_blocks((N, H, W, C), dev) if carrier is not None else (None, None)
        y8 = act8.empty_blocks((N, H, W, C), dev) if out8 else (None, None)
        ws = _bytes(_ws_bytes(N, H * W, C, G), dev)  # (held by its name until the launches are enqueued)
        with act8.on(dev):
            _lib.check(_lib.load().esr_gn_lrelu_fwd(x.data_ptr(), N, H * W, C, G, _p(gamma), _p(beta), eps, slope,
                                                    y.data_ptr(), stat.data_ptr(), _p(codes), _p(exps), _p(y8[0]),
                                                    _p(y8[1]), ws.data_ptr(), act8.stream(dev)), 'esr_gn_lrelu_fwd')
        ctx.save_for_backward(x if carrier is None else carrier, codes, exps, gamma, beta, stat)
        ctx.geom = (G, slope)
        ctx.set_materialize_grads(False)  # no gradients of zeros for y's blocks
        if not out8:
            return y
        ctx.mark_non_differentiable(*y8)
        return (y,) + y8

    @staticmethod
    def backward(ctx, gy, *_blocks):
        if gy is None:
            return (None,) * 8
        src, codes, exps, gamma, beta, stat = ctx.saved_tensors
        gy = _nhwc(gy)
        if torch.is_grad_enabled():
            gx, gg, gb = _GNLReLUBwdFn.apply(src, gamma, beta, gy, codes, exps, stat, *ctx.geom)
        else:
            gx, gg, gb, _ = _bwd(src, codes, exps, gamma, beta, stat, gy, *ctx.geom, False)
        return gx, None, gg if gamma is not None else None, gb if beta is not None else None, None, None, None, None


class _GNLReLUBwdFn(torch.autograd.Function):
    """(x, γ, gy) -> (gx, dγ, dβ) of the layer, differentiable once more (esr_gn_lrelu_bwd2)."""

    @staticmethod
    def forward(ctx, src, gamma, beta, gy, codes, exps, stat, G, slope):
        gx, gg, gb, sums = _bwd(src, codes, exps, gamma, beta, stat, gy, G, slope, True)
        ctx.save_for_backward(src, gamma, beta, gy, codes, exps, stat, sums)
        ctx.geom = (G, slope)
        ctx.set_materialize_grads(False)
        return gx, gg, gb

    @staticmethod
    def backward(ctx, ggx, ggg, ggb):
        if torch.is_grad_enabled():  # (once_differentiable lets autograd.grad go round its error to a wrong result)
            raise RuntimeError('group_norm_lrelu is differentiable twice: no graph of its second derivative '
                               '(create_graph) can be made')
        src, gamma, beta, gy, codes, exps, stat, sums = ctx.saved_tensors
        if ggx is None and ggg is None and ggb is None:
            return (None,) * 9
        G, slope = ctx.geom
        N, C, H, W = gy.shape
        dev = gy.device
        g_x, g_gy = torch.empty_like(gy), torch.empty_like(gy)
        g_gamma = torch.empty(C, device=dev, dtype=torch.float32) if gamma is not None else None
        ggx = None if ggx is None else _nhwc(ggx)
        ggg, ggb = (None if t is None else t.contiguous() for t in (ggg, ggb))
        ws = _bytes(_ws_bytes(N, H * W, C, G), dev)
        with act8.on(dev):
            _lib.check(_lib.load().esr_gn_lrelu_bwd2(_p(src) if codes is None else None, _p(codes), _p(exps),
                                                     gy.data_ptr(), _p(ggx), _p(ggg), _p(ggb), N, H * W, C, G,
                                                     _p(gamma), _p(beta), stat.data_ptr(), slope, sums.data_ptr(),
                                                     g_x.data_ptr(), g_gy.data_ptr(), _p(g_gamma), ws.data_ptr(),
                                                     act8.stream(dev)), 'esr_gn_lrelu_bwd2')
        return g_x, g_gamma, None, g_gy, None, None, None, None, None


def group_norm_lrelu(x, groups, weight=None, bias=None, eps=1e-5, slope=0.2, checkpoint=None, out8=False):
    """leaky_relu(group_norm(x, groups, weight, bias, eps), slope) of a float32 NCHW tensor with channels-last storage
    (another memory format is copied), differentiable twice in x, weight and the incoming gradient.  slope 1 is the norm
    alone, 0 a ReLU.  checkpoint='int8': x is kept for the backward in 8 bits, the slope taken at each value exactly.
    Returns an NCHW tensor with channels-last storage; out8: (that, its act8.Act8 blocks [N, H, W, C]) from the same
    pass, for a layer that keeps its input in 8 bits."""
    act8.check_mode(checkpoint)
    if x.dim() != 4:
        raise ValueError('group_norm_lrelu: an NCHW tensor, got %d dimensions' % x.dim())
    B, C, H, W = x.shape
    if groups < 1 or C % groups:
        raise ValueError('group_norm_lrelu: %d channels in %d groups' % (C, groups))
    if H * W == 0:
        raise ValueError('group_norm_lrelu: no values to normalise in %s' % (tuple(x.shape),))
    for t in (weight, bias):
        if t is not None and tuple(t.shape) != (C,):
            raise ValueError('group_norm_lrelu: weight and bias have %d values, got %s' % (C, tuple(t.shape)))
    if not (eps >= 0 and math.isfinite(eps) and math.isfinite(slope)):
        raise ValueError('group_norm_lrelu: eps %r, slope %r' % (eps, slope))
    dev = act8.check_dev('gn', x, weight, bias)
    if B == 0:
        y = x * 1.0
        for t in (weight, bias):  # (a gradient of zeros, as nn.GroupNorm's)
            y = y if t is None else y * t.view(1, C, 1, 1)
        return (y, act8.Act8(*act8.empty_blocks((0, H, W, C), dev), C)) if out8 else y
    x = _nhwc(x)
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    needs = checkpoint and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias))
    out = _GNLReLUFn.apply(x, act8.Carrier.apply(x) if needs else None, weight, bias, int(groups), float(eps),
                           float(slope), bool(out8))
    return (out[0], act8.Act8.of(*out[1:], (B, H, W, C))) if out8 else out


class HipGroupNorm(nn.GroupNorm):
    """nn.GroupNorm (same parameters, state_dict and init) of NCHW float32 tensors with channels-last storage, on HIP.
    discriminator._run fuses the LeakyReLU that follows it (`lrelu`)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, checkpoint=None):
        super().__init__(num_groups, num_channels, eps=eps, affine=affine)
        self.checkpoint = act8.check_mode(checkpoint)

    def check(self, x):
        """Refuses an input of one value per (sample, group), as nn.InstanceNorm2d does: what the layer gives is its bias
        then, whatever the value, and no gradient passes it."""
        if x.dim() == 4 and x.shape[2] * x.shape[3] * (self.num_channels // self.num_groups) == 1:
            raise ValueError('HipGroupNorm: one value per sample and group in %s, %d groups: its norm is 0 for every input'
                             % (tuple(x.shape), self.num_groups))

    def lrelu(self, x, slope, out8=False):
        self.check(x)
        return group_norm_lrelu(x, self.num_groups, self.weight, self.bias, self.eps, slope, self.checkpoint, out8)

    def forward(self, x):
        return self.lrelu(x, 1.0)
