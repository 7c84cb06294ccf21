"""GroupNorm + LeakyReLU of channels-last activations, fused on HIP (csrc/esr_gn.hip): forward, backward and the
backward's own backward, which the WGAN-GP penalty needs (loss.py:244-263).

The norm for a critic under a gradient penalty: the penalty bounds the gradient of each sample's score, and a batch norm
makes that score a function of the other samples.  Statistics are per (sample, group of channels), so a layer has no
running buffers, is the same in training and eval mode, and is the same on every rank.  One group per channel without
affine parameters is instance norm (block.py:46-58).  With checkpoint='int8' the layer keeps its input in 8 bits (act8.py)
instead of fp32 until its backward."""
import math

import torch
import torch.nn as nn

from . import _lib
from . import act8


def _p(t):
    return None if t is None else t.data_ptr()


def _ws(lib, x2, G):
    n = int(lib.esr_gn_workspace_bytes(x2.shape[0], x2.shape[1], x2.shape[2], G))
    if n < 0:
        raise RuntimeError('esr_gn_workspace_bytes failed with esr_status %d for [N, HW, C] = %s, %d groups'
                           % (n, tuple(x2.shape), G))
    return torch.empty(n, device=x2.device, dtype=torch.uint8)


class _GNLReLUFn(torch.autograd.Function):
    """[N, HW, C] -> lrelu(gn(x)).  `carrier` is None, or act8.Carrier's stand-in for x: then x is kept in 8 bits."""

    @staticmethod
    def forward(ctx, x2, carrier, gamma, beta, G, eps, slope):
        lib = _lib.load()
        N, HW, C = x2.shape
        y = torch.empty_like(x2)
        stat = torch.empty(N, G, 2, device=x2.device, dtype=torch.float64)
        codes, exps = act8.empty_blocks(x2.shape, x2.device) if carrier is not None else (None, None)
        with torch.cuda.device(x2.device):
            _lib.check(lib.esr_gn_lrelu_fwd(x2.data_ptr(), N, HW, C, G, _p(gamma), _p(beta), eps, slope, y.data_ptr(),
                                            stat.data_ptr(), _p(codes), _p(exps), _ws(lib, x2, G).data_ptr(),
                                            act8._stream(x2)), 'esr_gn_lrelu_fwd')
        ctx.save_for_backward(x2 if carrier is None else carrier, codes, exps, gamma, beta, stat)
        ctx.geom = (G, slope)
        return y

    @staticmethod
    def backward(ctx, gy):
        src, codes, exps, gamma, beta, stat = ctx.saved_tensors
        gx, gg, gb = _GNLReLUBwdFn.apply(src, gamma, beta, gy.contiguous(), codes, exps, stat, *ctx.geom)
        return gx, None, gg if gamma is not None else None, gb if beta is not None else None, None, None, None


class _GNLReLUBwdFn(torch.autograd.Function):
    """(x, γ, gy) -> (gx, dγ, dβ) of the layer, differentiable once more (esr_gn_lrelu_bwd2)."""

    @staticmethod
    def forward(ctx, src, gamma, beta, gy, codes, exps, stat, G, slope):
        lib = _lib.load()
        N, HW, C = gy.shape
        gx = torch.empty_like(gy)
        gg, gb = torch.empty(C, device=gy.device), torch.empty(C, device=gy.device)
        sums = torch.empty(N, 2, C, device=gy.device, dtype=torch.float64)
        with torch.cuda.device(gy.device):
            _lib.check(lib.esr_gn_lrelu_bwd(_p(src) if codes is None else None, _p(codes), _p(exps), gy.data_ptr(), N,
                                            HW, C, G, _p(gamma), _p(beta), stat.data_ptr(), slope, gx.data_ptr(),
                                            gg.data_ptr(), gb.data_ptr(), sums.data_ptr(), _ws(lib, gy, G).data_ptr(),
                                            act8._stream(gy)), 'esr_gn_lrelu_bwd')
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
        lib = _lib.load()
        N, HW, C = gy.shape
        g_x, g_gy = torch.empty_like(gy), torch.empty_like(gy)
        g_gamma = torch.empty(C, device=gy.device) if gamma is not None else None
        ggx, ggg, ggb = (None if t is None else t.contiguous() for t in (ggx, ggg, ggb))
        with torch.cuda.device(gy.device):
            _lib.check(lib.esr_gn_lrelu_bwd2(_p(src) if codes is None else None, _p(codes), _p(exps), gy.data_ptr(),
                                             _p(ggx), _p(ggg), _p(ggb), N, HW, C, G, _p(gamma), _p(beta),
                                             stat.data_ptr(), slope, sums.data_ptr(), g_x.data_ptr(), g_gy.data_ptr(),
                                             _p(g_gamma), _ws(lib, gy, G).data_ptr(), act8._stream(gy)),
                       'esr_gn_lrelu_bwd2')
        return g_x, g_gamma, None, g_gy, None, None, None, None, None


def group_norm_lrelu(x, groups, weight=None, bias=None, eps=1e-5, slope=0.2, checkpoint=None):
    """leaky_relu(group_norm(x, groups, weight, bias, eps), slope) of a float32 NCHW tensor with channels-last storage
    (another memory format is copied), differentiable twice in x, weight and the incoming gradient.  slope 1 is the norm
    alone, 0 a ReLU.  checkpoint='int8': x is kept for the backward in 8 bits, the slope taken at each value exactly.
    Returns an NCHW tensor with channels-last storage."""
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
    act8.check_dev('gn', x, weight, bias)
    if B == 0:
        return x * 1.0
    xh = x.permute(0, 2, 3, 1)
    if not xh.is_contiguous():
        xh = xh.contiguous()
    x2 = xh.view(B, H * W, C)
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    needs = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias))
    carrier = act8.Carrier.apply(x2) if checkpoint and needs else None
    y = _GNLReLUFn.apply(x2, carrier, weight, bias, int(groups), float(eps), float(slope))
    return y.view(B, H, W, C).permute(0, 3, 1, 2)


class HipGroupNorm(nn.GroupNorm):
    """nn.GroupNorm (same parameters, state_dict and init) of NCHW float32 tensors with channels-last storage, on HIP.
    discriminator._run fuses the LeakyReLU that follows it (`lrelu`)."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, checkpoint=None):
        super().__init__(num_groups, num_channels, eps=eps, affine=affine)
        self.checkpoint = act8.check_mode(checkpoint)

    def lrelu(self, x, slope):
        return group_norm_lrelu(x, self.num_groups, self.weight, self.bias, self.eps, slope, self.checkpoint)

    def forward(self, x):
        return self.lrelu(x, 1.0)
