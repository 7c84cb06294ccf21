"""Activations kept in 8 bits between the forward and the backward pass (csrc/esr_act8.hip).

A training step of the discriminator keeps every convolution's input and every norm's input until the backward reads
them: 8 bytes per activation value in fp32.  `pack` keeps 1 + 1/32: int8 codes that share a power-of-two step per 32
channels of a pixel (error <= half a step <= max|x|/127 of the block; x > 0 is kept exactly, so LeakyReLU masks are: a
positive value below half a step takes code 1).
The kernels of the weight gradients (dconv.conv_wgrad_act8) and of the norm's backward (gn.group_norm_lrelu with
checkpoint='int8') read the codes themselves; the first block's LeakyReLU mask, a convolution's second derivative and weight
gradients of another precision than x3 unpack them first."""
import contextlib

import torch

from . import _lib

BLOCK = 32
# what the `checkpoint` / `act_checkpoint` arguments of gn.py, dconv.py and discriminator.py take
CHECKPOINTS = (None, 'int8')


def check_mode(mode):
    if mode not in CHECKPOINTS:
        raise ValueError('act_checkpoint is one of %s, got %r' % (CHECKPOINTS, mode))
    return mode


_HERE = contextlib.nullcontext()


def on(dev):
    """The context in which launches go to `dev` (entering torch.cuda.device costs several launches' host time)."""
    return _HERE if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def stream(dev):
    """The current stream's handle (without the Stream object that torch.cuda.current_stream makes: 0.3 us for 2)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def check_dev(what, *ts):
    """The first tensor's device, after checking that every tensor (None skipped) is float32 and on it."""
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda or t.dtype != torch.float32:
            raise RuntimeError('esr_amd.%s: tensors must be float32 on a ROCm device (this build has no CPU path)' % what)
        dev = t.device if dev is None else dev
        if t.device != dev:
            raise RuntimeError('esr_amd.%s: tensors on %s and %s' % (what, dev, t.device))
    return dev


def pitch(C):
    """Codes of a pixel of C channels: rows of 16 bytes."""
    return -(-C // 16) * 16


def empty_blocks(shape, dev):
    """Unwritten (codes, exps) of an activation of `shape` [..., C]."""
    lead, C = tuple(shape[:-1]), shape[-1]
    return (torch.empty(lead + (pitch(C),), device=dev, dtype=torch.int8),
            torch.empty(lead + (-(-C // BLOCK),), device=dev, dtype=torch.uint8))


class Act8:
    """An activation of `shape` [..., C] in 8 bits: codes int8 [..., C rounded up to 16] and exps uint8
    [..., ceil(C / 32)]; the value of a code is code · 2^(e − 132), NaN where e = 255."""
    __slots__ = ('codes', 'exps', 'shape')

    def __init__(self, codes, exps, channels):
        lead = tuple(codes.shape[:-1])
        if codes.dtype != torch.int8 or exps.dtype != torch.uint8 or codes.dim() < 1 or channels < 1 or \
                codes.shape[-1] != pitch(channels) or tuple(exps.shape) != lead + (-(-channels // BLOCK),):
            raise ValueError('Act8: int8 codes [..., %d] with uint8 exponents [..., %d] for %d channels, got %s %s and %s %s'
                             % (pitch(channels), -(-channels // BLOCK), channels, codes.dtype, tuple(codes.shape),
                                exps.dtype, tuple(exps.shape)))
        if codes.device != exps.device:
            raise RuntimeError('Act8: codes on %s, exponents on %s' % (codes.device, exps.device))
        codes = codes.contiguous()
        self.codes = codes if codes.data_ptr() % 16 == 0 else codes.clone()
        self.exps, self.shape = exps.contiguous(), lead + (channels,)

    @classmethod
    def of(cls, codes, exps, shape):
        """Blocks that this package has just written, without the checks."""
        a = cls.__new__(cls)
        a.codes, a.exps, a.shape = codes, exps, tuple(shape)
        return a

    @property
    def nbytes(self):
        return self.codes.numel() + self.exps.numel()

    def unpack(self):
        """The values, float32 [..., C]."""
        if not self.codes.is_cuda:
            raise RuntimeError('esr_amd.act8: tensors must be on a ROCm device (this build has no CPU path)')
        x = torch.empty(self.shape, device=self.codes.device, dtype=torch.float32)
        if x.numel():
            with on(x.device):
                _lib.check(_lib.load().esr_act8_unpack(self.codes.data_ptr(), self.exps.data_ptr(),
                                                       x.numel() // self.shape[-1], self.shape[-1], x.data_ptr(),
                                                       stream(x.device)), 'esr_act8_unpack')
        return x


def pack(x):
    """Act8 of a float32 tensor [..., C] (channels last; a copy is made of one that is not contiguous).  Not
    differentiable: what the backward keeps, not an operation of the forward."""
    check_dev('act8', x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('act8.pack: a tensor [..., C], got %s' % (tuple(x.shape),))
    if not x.is_contiguous():
        x = x.detach().contiguous()
    codes, exps = empty_blocks(x.shape, x.device)
    if x.numel():
        with on(x.device):
            _lib.check(_lib.load().esr_act8_pack(x.data_ptr(), x.numel() // x.shape[-1], x.shape[-1], codes.data_ptr(),
                                                 exps.data_ptr(), stream(x.device)), 'esr_act8_pack')
    return Act8.of(codes, exps, x.shape)


class Carrier(torch.autograd.Function):
    """A tensor of x's shape that holds no values (all strides 0) and hands its gradient on to x: what a layer with an
    8-bit checkpoint saves in x's place, so that the backward's own backward finds its way to x without keeping x."""

    @staticmethod
    def forward(ctx, x):
        ctx.set_materialize_grads(False)  # a first-order backward has no gradient for it: not one of zeros either
        return torch.empty_strided(x.shape, (0,) * x.dim(), device=x.device, dtype=x.dtype)

    @staticmethod
    def backward(ctx, g):
        return g
