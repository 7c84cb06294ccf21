"""Memory handed to a launch is held until the call has returned: a workspace or a copy that only lives while the
arguments are evaluated goes back to the allocator before the launch is enqueued, and another thread's tensor (or the
next argument's) can be given the same memory.  The library is stubbed; the calls run on CPU tensors."""
import contextlib
import gc

import pytest
import torch

from esr_amd import _lib, act8, bn, gn


class Storages:
    """The storages that torch.empty and Tensor.contiguous hand out, by address.  They are kept, so that no address comes
    twice; one that nothing but this list holds has been released."""

    def __init__(self, monkeypatch):
        self.seen = {}
        for owner, name in ((torch, 'empty'), (torch.Tensor, 'contiguous')):
            self.wrap(monkeypatch, owner, name)

    def wrap(self, monkeypatch, owner, name):
        real = getattr(owner, name)

        def call(*a, **k):
            k.pop('device', None)
            t = real(*a, **k)
            self.seen[t.data_ptr()] = t.untyped_storage()
            return t
        monkeypatch.setattr(owner, name, call)

    def released(self, p):
        return p in self.seen and torch._C._storage_Use_Count(self.seen[p]._cdata) == 1


class Stub:
    """Every entry point returns 0 after checking that the pointers among its arguments belong to living tensors."""

    def __init__(self, storages):
        self.storages, self.calls = storages, []

    def __getattr__(self, name):
        if not name.startswith('esr_'):
            raise AttributeError(name)

        def entry(*args):
            gc.collect()
            for i, a in enumerate(args):
                assert not (isinstance(a, int) and self.storages.released(a)), \
                    '%s: the memory of argument %d was released before the launch' % (name, i)
            self.calls.append((name, args))
            return 1 << 10 if name.endswith(('_bytes', '_floats', '_blocks')) else 0
        return entry


@pytest.fixture
def stub(monkeypatch):
    lib = Stub(Storages(monkeypatch))
    monkeypatch.setattr(_lib, 'load', lambda: lib)
    monkeypatch.setattr(act8, 'on', lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(act8, 'stream', lambda dev: 0)
    monkeypatch.setattr(bn, '_stream', lambda t: None)
    monkeypatch.setattr(act8, 'check_dev', lambda what, *ts: ts[0].device)
    gn._ws_bytes.cache_clear()
    yield lib
    gn._ws_bytes.cache_clear()  # the stub's sizes


@pytest.mark.parametrize('ck', [None, 'int8'])
@pytest.mark.parametrize('out8', [False, True])
def test_group_norm_workspaces(stub, ck, out8):
    x = torch.randn(2, 8, 4, 4).contiguous(memory_format=torch.channels_last).requires_grad_()
    w, b = torch.ones(8, requires_grad=True), torch.zeros(8, requires_grad=True)
    y = gn.group_norm_lrelu(x, 4, w, b, checkpoint=ck, out8=out8)
    y = y[0] if out8 else y
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b), create_graph=True)
    torch.autograd.grad(gx.sum() + gw.sum() + gb.sum(), (x, w))
    assert [n for n, _ in stub.calls if 'lrelu' in n] == ['esr_gn_lrelu_fwd', 'esr_gn_lrelu_bwd', 'esr_gn_lrelu_bwd2']


def test_batch_norm_workspaces(stub):
    """bn_lrelu, with upstream gradients of dγ and dβ that are expanded scalars: their copies live as long (released while
    the arguments were evaluated, dβ's took dγ's memory)."""
    m = torch.nn.BatchNorm2d(8)
    x = torch.randn(2, 8, 4, 4).contiguous(memory_format=torch.channels_last).requires_grad_()
    gx, gw, gb = torch.autograd.grad(bn.bn_lrelu(x, m, 0.2).sum(), (x, m.weight, m.bias), create_graph=True)
    torch.autograd.grad(gx.sum() + 2 * gw.sum() + 3 * gb.sum(), (x, m.weight))
    assert [n for n, _ in stub.calls if 'lrelu' in n] == ['esr_bn_lrelu_fwd', 'esr_bn_lrelu_bwd', 'esr_bn_lrelu_bwd2']


def test_first_block_and_cem_filters(stub, monkeypatch):
    """Weights and filters that are not contiguous (a network moved to channels last, a transposed filter) are copied; the
    copies live until the launches are enqueued."""
    from esr_amd import cem_ops, dconv, engine
    for m in (dconv, cem_ops):
        monkeypatch.setattr(m, '_stream', lambda t: None)
    monkeypatch.setattr(cem_ops, '_check', lambda *ts: None)
    monkeypatch.setattr(engine, '_require_device', lambda *a: None)
    w = torch.randn(64, 3, 3, 3).to(memory_format=torch.channels_last)
    x, gy = torch.randn(1, 6, 5, 3), torch.randn(1, 6, 5, 64)
    dconv._df_fwd(x, w, None, 0.2, 1)
    dconv._df_bwd(x, gy, gy, 0.2, w, True, True)
    f, img = torch.randn(7, 7).t(), torch.randn(3, 16, 16)
    cem_ops.downscale(img, f, 4)
    cem_ops.upscale(img, f, 4)
    cem_ops.filter_same(img, f)

    def layer():
        op = type('Op', (), {})()
        op.Filter_OP = type('Filter', (), {'weight': torch.randn(3, 1, 7, 7).transpose(2, 3)})()
        return op
    cem = type('Cem', (), {'DownscaleOP': layer(), 'Conv_LR_with_Inv_hTh_OP': layer(), 'Upscale_OP': layer()})()
    engine.cem_apply(stub, cem, torch.randn(1, 3, 32, 32), torch.randn(1, 3, 8, 8), 1, 8, 8, 0, None)
    names = [n for n, _ in stub.calls]
    want = {'dfirst_fwd': 1, 'dfirst_bwd': 1, 'cem_down': 2, 'cem_inv': 2, 'cem_up_add': 2}
    assert {n: names.count('esr_' + n) for n in want} == want


@pytest.mark.parametrize('ck', [None, 'int8'])
def test_blocks_get_no_gradients_of_zeros(stub, monkeypatch, ck):
    """Layers that hand on their output's 8-bit blocks beside it: the backward makes no gradient for them (zeros of their
    size in every backward)."""
    from torch.profiler import ProfilerActivity, profile

    from esr_amd import dconv
    monkeypatch.setattr(dconv, '_stream', lambda t: None)
    monkeypatch.setattr(dconv, '_check_dev', lambda *ts: None)
    monkeypatch.setattr(act8.Act8, 'unpack', lambda self: torch.empty(self.shape))
    x = torch.randn(2, 8, 4, 4).contiguous(memory_format=torch.channels_last).requires_grad_()
    y, _ = gn.group_norm_lrelu(x, 4, checkpoint=ck, out8=True)
    outs = [(y, x)]
    if ck:
        conv = dconv.HipConv2d(3, 64, 3, padding=1)
        conv.act_checkpoint = ck
        img = torch.randn(1, 3, 6, 5).contiguous(memory_format=torch.channels_last).requires_grad_()
        outs.append((dconv.dfirst_lrelu8(img, conv, 0.2)[0], img))
    for out, leaf in outs:
        gy = torch.randn_like(out)
        with profile(activities=[ProfilerActivity.CPU]) as prof:
            torch.autograd.grad(out, leaf, gy)
        names = {e.name for e in prof.events()}
        assert not names & {'aten::zeros', 'aten::zeros_like'}, names
