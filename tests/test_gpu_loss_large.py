'''linear_cross_entropy where one dimension of a launch does not hold the workgroups: more than 2^32 threads for the
logits' tiles, and for the rows of the hidden states' gradient.'''
import pytest
import torch

from loss_ref import ce64, check

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF = torch.bfloat16


def test_logit_tiles():
    '''2^22 + 128 rows of 2^17 words: 2^24 + 2^9 tiles of 256 threads.  The rows repeat after 64, so one small reference serves them all.'''
    from motif.ops import linear_cross_entropy
    N, d, V = 2 ** 22 + 128, 8, 2 ** 17
    g = torch.Generator(device=DEV).manual_seed(1)
    base = torch.randn(64, d, generator=g, device=DEV).to(BF)
    w = torch.randn(V, d, generator=g, device=DEV).to(BF)
    labels = torch.randint(0, V, (64,), generator=g, device=DEV)
    labels[5] = -100
    loss = linear_cross_entropy(base.repeat(N // 64, 1), w, labels.repeat(N // 64), reduction='none')
    want, tol = ce64(base, w, labels, reduction='none')
    check(loss.view(-1, 64), want.expand(N // 64, 64), tol.expand(N // 64, 64), 'loss')


def test_gradient_rows():
    '''2^23 rows of 513 features: a thread for each feature of nine waves a row.'''
    from motif.ops import linear_cross_entropy
    N, d, V = 2 ** 23, 513, 2
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(N, d, generator=g, device=DEV, dtype=BF).requires_grad_()
    w = torch.randn(V, d, generator=g, device=DEV).mul(0.1).to(BF)
    labels = torch.randint(-1, V, (N,), generator=g, device=DEV)
    one = torch.ones((), device=DEV)
    loss = linear_cross_entropy(x, w, labels, ignore_index=-1, reduction='sum')
    dx, = torch.autograd.grad(loss, x, one)
    for at in (0, 2 ** 22, N - 2000):
        rows = slice(at, at + 2000)
        ref = ce64(x[rows], w, labels[rows], one, 'sum', ignore=-1)
        check(dx[rows], ref[2], ref[3], f'dx from row {at}')
