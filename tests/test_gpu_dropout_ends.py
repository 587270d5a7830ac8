'''dropout_add at the upper end of p, at an element whose word is all ones: element 30338 under the key 149059.'''
import pytest
import torch

from loss_ref import kept

pytestmark = pytest.mark.gpu

DEV = 'cuda'
SEED, AT, N = 149059, 30338, 30400
DTYPES = pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32], ids=['bf16', 'fp16', 'fp32'])


def test_the_word():
    '''T = 2^32 - 1 keeps that element alone.'''
    keep = kept(N, SEED, 1 - 2.0 ** -32)
    assert keep.nonzero().tolist() == [[AT]] and not kept(N, SEED, 1 - 2.0 ** -33).any()


@DTYPES
@pytest.mark.parametrize('p', [1 - 2.0 ** -33, 1 - 2.0 ** -40, 1 - 2.0 ** -53])
def test_a_threshold_above_every_word_keeps_none(p, dtype):
    '''round(p 2^32) = 2^32.'''
    from motif.ops import dropout_add
    x = torch.full((N,), 2.0, device=DEV, dtype=dtype)
    x[AT] = float('inf')
    res = torch.arange(N, device=DEV).to(dtype)
    for seed in (SEED, torch.tensor([SEED], device=DEV)):
        xg, rg = x.clone().requires_grad_(), res.clone().requires_grad_()
        y = dropout_add(xg, p, seed)
        assert not y.any()
        assert not torch.autograd.grad(y, xg, torch.ones_like(x))[0].any()
        y = dropout_add(xg, p, seed, residual=rg)
        assert torch.equal(y, res)
        dx, dr = torch.autograd.grad(y, (xg, rg), x)
        assert not dx.any() and torch.equal(dr, x)


def test_the_highest_threshold_that_a_word_reaches():
    from motif.ops import dropout_add
    x = torch.ones(N, device=DEV)
    y = dropout_add(x, 1 - 2.0 ** -32, SEED)
    assert y.nonzero().tolist() == [[AT]] and float(y[AT]) == 2.0 ** 32
