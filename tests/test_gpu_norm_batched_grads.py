'''Several gradients at once (is_grads_batched, a vectorised jacobian) through RMSNorm and the row norms, as through torch's own
op: each equals the gradient taken alone.'''
import pytest
import torch

from support import gen

pytestmark = pytest.mark.gpu

DEV = 'cuda'
U = 2.0 ** -24


def _layer(x, w, b):
    from motif.ops import layer_norm_rows
    return layer_norm_rows(x, w, b, 1e-5)


def _rms(x, w, b):
    from motif.ops import rms_norm_rows
    return rms_norm_rows(x, w, 1e-5)


def _module(x, w, b):
    from motif.ops.rms_norm import _rms
    return _rms(x, w, 1e-5)


@pytest.mark.parametrize('f,leaves', [(_module, 2), (_rms, 2), (_layer, 3)])
@pytest.mark.parametrize('shape', [(7, 40), (2, 3, 16), (24,)])
def test_batched_gradients(f, leaves, shape):
    g = gen(1)
    D = shape[-1]
    ins = [torch.randn(s, generator=g).to(DEV).requires_grad_() for s in (shape, (D,), (D,))]
    y = f(*ins)
    dys = torch.randn(5, *shape, generator=g).to(DEV)
    got = torch.autograd.grad(y, ins[:leaves], dys, is_grads_batched=True, retain_graph=True)
    alone = [torch.autograd.grad(y, ins[:leaves], dy, retain_graph=True) for dy in dys]
    for i, a in enumerate(got):
        want = torch.stack([one[i] for one in alone])
        # both in fp32: two sums of D (or of the rows) terms each and a dozen operations, of the largest entry's size
        assert a.shape == want.shape and (a - want).abs().max() <= 2 * (D + 24) * U * want.abs().max()


def test_a_vectorised_jacobian_of_the_module():
    from motif.ops import RMSNorm
    norm = RMSNorm(12).to(DEV)
    x = torch.randn(3, 12, generator=gen(2)).to(DEV)
    want = torch.autograd.functional.jacobian(norm, x)
    got = torch.autograd.functional.jacobian(norm, x, vectorize=True)
    assert (got - want).abs().max() <= 2 * 36 * U * want.abs().max()
