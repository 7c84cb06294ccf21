"""Derivatives of every order of the convolution that keeps its input in 8 bits (dconv.DConvAct8Fn), in float64 on the
CPU: the kernels are replaced by PyTorch's convolution, and the input's values are ones that its blocks hold exactly, so
that every derivative is the plain convolution's."""
import pytest
import torch
import torch.nn.functional as F

from esr_amd import act8, dconv

nchw = lambda t: t.permute(0, 3, 1, 2)  # noqa: E731
nhwc = lambda t: t.permute(0, 2, 3, 1).contiguous()  # noqa: E731


@pytest.fixture
def plain(monkeypatch):
    def unpack(self):
        step = torch.exp2(self.exps.double() - 132).repeat_interleave(32, -1)
        return self.codes[..., :self.shape[-1]].double() * step[..., :self.shape[-1]]

    def wgrad(x, gy, k, s, p, prec=None):
        return torch.nn.grad.conv2d_weight(nchw(x), (gy.shape[3], x.shape[3], k, k), nchw(gy), s, p)
    monkeypatch.setattr(act8.Act8, 'unpack', unpack)
    monkeypatch.setattr(dconv, 'conv_forward',
                        lambda x, w, b, k, s, p, prec=None: nhwc(F.conv2d(nchw(x), w, b, s, p)))
    monkeypatch.setattr(dconv, 'conv_dgrad', lambda gy, w, k, s, p, H, W, prec=None: nhwc(
        torch.nn.grad.conv2d_input((gy.shape[0], w.shape[1], H, W), w, nchw(gy), s, p)))
    monkeypatch.setattr(dconv, 'conv_wgrad', wgrad)
    monkeypatch.setattr(dconv, 'conv_wgrad_act8', lambda x8, gy, k, s, p: wgrad(x8.unpack(), gy, k, s, p))
    monkeypatch.setattr(dconv, '_bias_grad', lambda gy: gy.sum((0, 1, 2)))


@pytest.mark.parametrize('k,s,p', [(3, 1, 1), (4, 2, 1)])
def test_orders(plain, k, s, p):
    g = torch.Generator().manual_seed(k)
    rnd = lambda *sh: torch.randn(*sh, generator=g, dtype=torch.float64).requires_grad_()  # noqa: E731
    shape = (2, 8, 9, 5)
    codes = torch.randint(-127, 128, shape[:3] + (16,), generator=g, dtype=torch.int8)
    codes[..., 5:] = 0
    exps = torch.randint(128, 136, shape[:3] + (1,), generator=g, dtype=torch.uint8)
    x0 = act8.Act8(codes, exps, 5).unpack()
    w0, b0 = rnd(7, 5, k, k), rnd(7)
    gy0 = rnd(2, dconv.out_size(8, k, s, p), dconv.out_size(9, k, s, p), 7)
    ups = [rnd(*sh) for sh in (shape, w0.shape, b0.shape)]
    ups2 = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (x0, w0, gy0)]

    def orders(conv):
        x, w, b, gy = (t.detach().clone().requires_grad_() for t in (x0, w0, b0, gy0))
        u = [t.detach().clone().requires_grad_() for t in ups]
        y = conv(x, w, b)
        first = torch.autograd.grad(y, (x, w, b), gy, create_graph=True)
        second = torch.autograd.grad(sum((a * v).sum() for a, v in zip(first, u)), (x, w, gy), create_graph=True)
        third = torch.autograd.grad(sum((a * v).sum() for a, v in zip(second, ups2)), [x, w, gy] + u, allow_unused=True,
                                    create_graph=True)
        return [y] + [torch.zeros(()).double() if t is None else t for t in first + second + third]
    want = orders(lambda x, w, b: nhwc(F.conv2d(nchw(x), w, b, s, p)))
    for conv in (lambda x, w, b: dconv.DConvFn.apply(x, w, b, k, s, p),
                 lambda x, w, b: dconv.DConvAct8Fn.apply(x, act8.Carrier.apply(x), codes, exps, w, b, k, s, p)):
        for i, (a, r) in enumerate(zip(orders(conv), want)):
            torch.testing.assert_close(a, r, rtol=1e-12, atol=1e-12 * float(r.detach().abs().max()),
                                       msg=lambda m, i=i: '%d: %s' % (i, m))


def test_weight_gradient_call_refuses_to_lose_a_gradient():
    x8 = act8.Act8(torch.zeros(1, 4, 4, 16, dtype=torch.int8), torch.zeros(1, 4, 4, 1, dtype=torch.uint8), 8)
    gy = torch.zeros(1, 4, 4, 8, requires_grad=True)
    with pytest.raises(RuntimeError, match='no derivative'):
        dconv.conv_wgrad_act8(x8, gy, 3, 1, 1)
    with pytest.raises(RuntimeError, match='ROCm device'):
        dconv.conv_wgrad_act8(x8, gy.detach(), 3, 1, 1)
    with torch.no_grad(), pytest.raises(RuntimeError, match='ROCm device'):
        dconv.conv_wgrad_act8(x8, gy, 3, 1, 1)


@pytest.mark.parametrize('prec,kernel', [(None, 'act8'), ('x3', 'act8'), ('x6', 'x6'), ('f32', 'f32')])
def test_precision_of_the_weight_gradient(plain, monkeypatch, prec, kernel):
    """A layer (or the module) set to another arithmetic than x3 has it for the weight gradient of its blocks too."""
    ran = []
    gw = torch.ones(4, 5, 3, 3, dtype=torch.float64)
    monkeypatch.setattr(dconv, 'conv_wgrad', lambda x, gy, k, s, p, prec=None: ran.append(prec) or gw)
    monkeypatch.setattr(dconv, 'conv_wgrad_act8', lambda x8, gy, k, s, p: ran.append('act8') or gw)
    x = torch.ones(1, 6, 6, 5, dtype=torch.float64)
    codes, exps = torch.ones(1, 6, 6, 16, dtype=torch.int8), torch.full((1, 6, 6, 1), 132, dtype=torch.uint8)
    w = torch.ones(4, 5, 3, 3, dtype=torch.float64, requires_grad=True)
    dconv.DConvAct8Fn.apply(x, x, codes, exps, w, None, 3, 1, 1, prec).sum().backward()
    assert ran == [kernel]
    if prec:
        prev = dconv.set_precision(prec)
        try:
            dconv.DConvAct8Fn.apply(x, x, codes, exps, w, None, 3, 1, 1).sum().backward()
        finally:
            dconv.set_precision(prev)
        assert ran == [kernel] * 2
