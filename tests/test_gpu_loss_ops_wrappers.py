'''Tensor subclasses that hold no memory of their own (as distributed tensors) are refused by the norms, dropout and the loss:
their null pointers must not stand for an argument left out.'''
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'


class Wrapper(torch.Tensor):
    '''The sizes of a tensor that is kept beside it.'''

    @staticmethod
    def __new__(cls, held):
        t = torch.Tensor._make_wrapper_subclass(cls, held.shape, strides=held.stride(), dtype=held.dtype, device=held.device)
        t.held = held
        return t

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError('no operations')


def _args():
    x = torch.linspace(-1, 1, 96, device=DEV).view(6, 16)
    return {'x': x, 'weight': torch.full((16,), 2.0, device=DEV), 'bias': torch.ones(16, device=DEV), 'residual': x + 1,
            'seed': torch.tensor([5], device=DEV), 'words': torch.ones(9, 16, device=DEV), 'labels': torch.arange(6, device=DEV)}


def _rms(a):
    from motif.ops import rms_norm_rows
    return rms_norm_rows(a['x'], a['weight'])


def _layer(a):
    from motif.ops import layer_norm_rows
    return layer_norm_rows(a['x'], a['weight'], a['bias'])


def _dropout(a):
    from motif.ops import dropout_add
    return dropout_add(a['x'], 0.5, a['seed'], residual=a['residual'])


def _loss(a):
    from motif.ops import linear_cross_entropy
    return linear_cross_entropy(a['x'], a['words'], a['labels'])


@pytest.mark.parametrize('op,name', [(_rms, 'x'), (_rms, 'weight'), (_layer, 'x'), (_layer, 'weight'), (_layer, 'bias'), (_dropout, 'x'),
                                     (_dropout, 'residual'), (_dropout, 'seed'), (_loss, 'x'), (_loss, 'words'), (_loss, 'labels')])
def test_refused(op, name):
    args = _args()
    op(args)
    args[name] = Wrapper(args[name])
    assert args[name].data_ptr() == 0
    with pytest.raises((ValueError, RuntimeError), match='no memory|no operations'):
        op(args)


@pytest.mark.parametrize('op', [_rms, _layer, _dropout, _loss])
def test_a_subclass_with_memory(op):
    class Named(torch.Tensor):
        pass
    args = _args()
    want = op(args)
    assert torch.equal(op({k: v.as_subclass(Named) for k, v in args.items()}).as_subclass(torch.Tensor), want)
