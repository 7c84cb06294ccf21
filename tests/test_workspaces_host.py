"""Memory handed to a launch is held until the call has returned: a workspace or a copy that only lives while the
arguments are evaluated goes back to the allocator before the launch is enqueued, and another thread's tensor (or the
next argument's) can be given the same memory.  The library is stubbed; the calls run on CPU tensors."""
import contextlib
import gc
import weakref

import pytest
import torch

from esr_amd import _lib, act8, bn, gn


class Storages:
    """Weak references to the tensors that torch.empty and Tensor.contiguous hand out, by address; the storages are kept,
    so that no address comes twice."""

    def __init__(self, monkeypatch):
        self.seen, self.kept = [], []
        for owner, name in ((torch, 'empty'), (torch.Tensor, 'contiguous')):
            self.wrap(monkeypatch, owner, name)

    def wrap(self, monkeypatch, owner, name):
        real = getattr(owner, name)

        def call(*a, **k):
            k.pop('device', None)
            t = real(*a, **k)
            self.seen.append((t.data_ptr(), weakref.ref(t)))
            self.kept.append(t.untyped_storage())
            return t
        monkeypatch.setattr(owner, name, call)


class Stub:
    """Every entry point returns 0 after checking that the pointers among its arguments belong to living tensors."""

    def __init__(self, storages):
        self.storages, self.calls = storages, []

    def __getattr__(self, name):
        def entry(*args):
            gc.collect()
            living = {p for p, r in self.storages.seen if r() is not None}
            known = {p for p, _ in self.storages.seen if p}
            for i, a in enumerate(args):
                if isinstance(a, int) and a in known:
                    assert a in living, '%s: the memory of argument %d was released before the launch' % (name, i)
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
    stub.storages.seen.clear()  # (its parameters are other objects on the memory that torch.empty gave)
    x = torch.randn(2, 8, 4, 4).contiguous(memory_format=torch.channels_last).requires_grad_()
    gx, gw, gb = torch.autograd.grad(bn.bn_lrelu(x, m, 0.2).sum(), (x, m.weight, m.bias), create_graph=True)
    torch.autograd.grad(gx.sum() + 2 * gw.sum() + 3 * gb.sum(), (x, m.weight))
    assert [n for n, _ in stub.calls if 'lrelu' in n] == ['esr_bn_lrelu_fwd', 'esr_bn_lrelu_bwd', 'esr_bn_lrelu_bwd2']
