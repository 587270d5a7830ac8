'''Gradients of the row norms taken under create_graph, where one input of the norm depends on another: the first
gradients are those of a plain backward, and second derivatives agree with float64 torch ops.'''
import pytest
import torch

from support import gen

pytestmark = pytest.mark.gpu

DEV = 'cuda'
N, D = 12, 40
# A pass over a row is off by (D + 12) 2^-24 = 3e-6 of its sizes; a gradient through two norms holds four such passes, its
# derivative some ten: 3e-5 of the largest entry, and a factor of three.
TOL = 1e-4


def _plain(x, w, b=None):
    c = x if b is None else x - x.mean(-1, keepdim=True)
    y = c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5) * w
    return y if b is None else y + b


def _kernels(x, w, b=None):
    from motif.ops import layer_norm_rows, rms_norm_rows
    return rms_norm_rows(x, w, 1e-5) if b is None else layer_norm_rows(x, w, b, 1e-5)


CASES = {
    'a weight used twice': lambda norm, x, w: norm(torch.tanh(norm(x, w)), w),
    'a weight from the input': lambda norm, x, w: norm(x, w * x.mean(0)),
    'an input from the weight': lambda norm, x, w: norm(x * w, w),
    'the weight as the bias': lambda norm, x, w: norm(x, w, w),
    'two layer norms of one weight': lambda norm, x, w: norm(torch.tanh(norm(x, w, w * x[0])), w, x.mean(0)),
}


def _grads(norm, f, x, w, dy):
    '''First gradients under create_graph, those of a plain backward, and second derivatives.'''
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    first = torch.autograd.grad(f(norm, x, w), (x, w), dy, create_graph=True)
    plain = torch.autograd.grad(f(norm, x, w), (x, w), dy)
    second = torch.autograd.grad(sum(g.square().sum() for g in first), (x, w))
    return [*first, *plain, *second]


@pytest.mark.parametrize('case', CASES)
def test_inputs_that_depend_on_each_other(case):
    g = gen(3)
    x, w, dy = (torch.randn(s, generator=g).to(DEV) for s in ((N, D), (D,), (N, D)))
    got = _grads(_kernels, CASES[case], x, w, dy)
    want = _grads(_plain, CASES[case], x.double(), w.double(), dy.double())
    names = ('dx', 'dw', 'plain dx', 'plain dw', 'second x', 'second w')
    for what, a, b in zip(names, got, want):
        off, size = float((a.double() - b).abs().max().detach()), float(b.abs().max().detach())
        assert off <= TOL * size, f'{what}: off by {off:.3g} of {size:.3g}'


def test_norm_module_shared_by_two_layers():
    '''A gradient penalty through an RMSNorm module that two layers share.'''
    from motif.ops import RMSNorm
    norm = RMSNorm(D).to(DEV)
    g = gen(4)
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(DEV)
    with torch.no_grad():
        norm.weight.copy_(w)
    x = torch.randn(N, D, generator=g).to(DEV).requires_grad_()

    def penalty(f, x, leaf):
        first = torch.autograd.grad(f(torch.tanh(f(x))).square().sum(), (x, leaf), create_graph=True)
        return (*first, *torch.autograd.grad(sum(d.square().sum() for d in first), (x, leaf)))
    got = penalty(norm, x, norm.weight)
    x64, w64 = x.detach().double().requires_grad_(), w.double().requires_grad_()
    eps = norm.eps
    want = penalty(lambda t: t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * w64, x64, w64)
    for a, b in zip(got, want):
        assert (a.double() - b).abs().max() <= TOL * b.abs().max()
