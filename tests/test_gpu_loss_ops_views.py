'''Tensors whose sign is applied when they are read (torch's negative views) go into the norms, dropout and the loss with it.'''
import pytest
import torch

from support import gen

pytestmark = pytest.mark.gpu

DEV = 'cuda'


def _neg(t):
    '''-t as a view of t's memory.'''
    v = torch._neg_view(t)
    assert v.is_neg() and v.data_ptr() == t.data_ptr()
    return v


def _rms(x, w, b, dy):
    from motif.ops import rms_norm_rows
    return rms_norm_rows(x, w)


def _layer(x, w, b, dy):
    from motif.ops import layer_norm_rows
    return layer_norm_rows(x, w, b)


def _module(x, w, b, dy):
    from motif.ops.rms_norm import _rms
    return _rms(x, w, 1e-6)


def _dropout(x, w, b, dy):
    from motif.ops import dropout_add
    return dropout_add(x, 0.25, 6, residual=dy)


def _loss(x, w, b, dy):
    from motif.ops import linear_cross_entropy
    return linear_cross_entropy(x, dy, torch.arange(len(x), device=x.device), reduction='none')


@pytest.mark.parametrize('op', [_rms, _layer, _module, _dropout, _loss])
@pytest.mark.parametrize('which', ['x', 'w', 'b', 'res', 'gradient'])
@pytest.mark.parametrize('grad', [True, False], ids=['training', 'inference'])
def test_negative_views(op, which, grad):
    '''One of the inputs, or the gradient that comes in, as such a view, against the same negated in memory.'''
    g = gen(1)
    ins = [torch.randn(s, generator=g).to(DEV) for s in ((20, 64), (64,), (64,), (20, 64))]

    def run(neg):
        leaves = [t.clone().requires_grad_(grad) for t in ins]
        y = op(*(neg(t) if name == which else t for name, t in zip(('x', 'w', 'b', 'res'), leaves)))
        if not grad:
            return [y]
        up = torch.linspace(-1, 1, y.numel(), device=DEV).view(y.shape)
        return [y.detach(), *torch.autograd.grad(y, leaves, neg(up) if which == 'gradient' else up, allow_unused=True)]
    got, want = run(_neg), run(torch.neg)
    assert len(got) == len(want)
    for a, c in zip(got, want):
        assert (a is None) == (c is None)
        assert a is None or bool((a == c).all())


def test_imaginary_parts_of_rows_of_one_feature():
    '''Such views come from conjugates; with one feature a row their strides are regular.'''
    from motif.ops import dropout_add, rms_norm_rows
    z = torch.complex(torch.randn(9, 1, generator=gen(2)), torch.randn(9, 1, generator=gen(3))).to(DEV)
    x = z.conj().imag
    assert x.is_neg()
    assert torch.equal(rms_norm_rows(x), rms_norm_rows(-z.imag)) and torch.equal(dropout_add(x, 0.0, 1), -z.imag)


@pytest.mark.parametrize('op', [_rms, _layer, _module, _dropout, _loss])
def test_zero_tensors(op):
    '''torch's zeros without memory (they come up in its derivatives), as an input and as the gradient that comes in.'''
    g = gen(4)
    x, w, b, res = (torch.randn(s, generator=g).to(DEV) for s in ((20, 64), (64,), (64,), (20, 64)))
    zero = torch._efficientzerotensor((20, 64), device=DEV)
    assert torch.equal(op(x, w, b, zero), op(x, w, b, torch.zeros_like(x)))
    assert torch.equal(op(zero, w, b, res), op(torch.zeros_like(x), w, b, res))
    leaf = x.clone().requires_grad_()
    y = op(leaf, w, b, res)
    dx, = torch.autograd.grad(y, leaf, torch._efficientzerotensor(tuple(y.shape), device=DEV))
    assert dx.shape == x.shape and not dx.any()
