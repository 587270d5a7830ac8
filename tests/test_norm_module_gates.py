'''RMSNorm in training where the autograd nodes' library does not load: torch's own op, with a warning.'''
import sys

import pytest
import torch
import torch.nn.functional as F

import motif
from motif.ops import RMSNorm, _lib, rms_norm

DEV = 'cuda'


@pytest.fixture
def without_nodes(monkeypatch):
    '''As if _autograd_nodes could not be imported.'''
    monkeypatch.delattr(motif, '_autograd_nodes', raising=False)
    monkeypatch.setitem(sys.modules, 'motif._autograd_nodes', None)
    monkeypatch.setattr(_lib, '_nodes', None)
    monkeypatch.setattr(_lib, '_nodes_found', None, raising=False)


def test_nodes_that_cannot_be_loaded(without_nodes, monkeypatch):
    monkeypatch.setattr(_lib, 'available', lambda: True)
    with pytest.raises(RuntimeError, match='autograd nodes'):
        _lib.nodes()
    x, w = torch.randn(3, 8, requires_grad=True), torch.ones(8)
    with pytest.warns(UserWarning, match='autograd nodes'):
        assert not rms_norm._trains_on_kernels(x, w)
    assert not rms_norm._trains_on_kernels(x, w) and not _lib.nodes_available()


def test_nodes_that_can(monkeypatch):
    monkeypatch.setattr(_lib, 'available', lambda: True)
    x, w = torch.randn(3, 8, requires_grad=True), torch.ones(8)
    assert rms_norm._trains_on_kernels(x, w) and _lib.nodes_available()
    monkeypatch.setattr(_lib, 'available', lambda: False)
    assert not rms_norm._trains_on_kernels(x, w) and not _lib.nodes_available()


def _train(norm, x, dy):
    x = x.detach().requires_grad_()
    y = norm(x)
    return (y.detach(), *torch.autograd.grad(y, (x, norm.weight), dy))


@pytest.mark.gpu
@pytest.mark.filterwarnings('ignore:the motif autograd nodes')
def test_training_without_the_nodes(without_nodes):
    norm = RMSNorm(64).to(DEV)
    x, dy = torch.randn(10, 64, device=DEV), torch.randn(10, 64, device=DEV)
    got = _train(norm, x, dy)
    want = _train(_Torch(norm), x, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match='autograd nodes'):
        from motif.ops import rms_norm_rows
        rms_norm_rows(x, norm.weight)


class _Torch:
    def __init__(self, norm):
        self.weight, self.eps = norm.weight, norm.eps

    def __call__(self, x):
        return F.rms_norm(x, self.weight.shape, self.weight, self.eps)
