'''A mask beside a window may leave a row of the materialised route no key: it gives zeros, as on
the kernels, and no other row hears of it.'''
import pytest
import torch

from motif.block.attention.chord_attn import ChordAttention
from support import gen


def _layers(n, **kw):
    torch.manual_seed(0)
    layers = [ChordAttention(hidden_size=64, num_heads=4, num_kv_heads=2, **kw).double().eval() for _ in range(n)]
    with torch.no_grad():
        for layer in layers:
            layer.theta_alpha.normal_(std=0.3)
            layer.theta_beta.normal_(std=0.2)
    return layers


def _stack(layers, x, mask=None):
    for layer in layers:
        x = x + layer(x, attention_mask=mask).output
    return x


def _x(B, L, seed=0):
    return torch.randn(B, L, 64, generator=gen(seed), dtype=torch.float64)


def _mask(kind, keep):
    if kind == 'bool':
        return keep
    return torch.zeros(keep.shape, dtype=torch.float64).masked_fill(~keep, float('-inf'))


@pytest.mark.parametrize('kind', ['bool', 'additive'])
@pytest.mark.parametrize('window,sinks', [(4, 0), (1, 0), (3, 2)])
@torch.no_grad()
def test_right_padding_longer_than_the_window(kind, window, sinks):
    layers, x, n = _layers(3, window=window, sinks=sinks), _x(2, 16), 8
    keep = (torch.arange(16) < n)[None, None, None].expand(2, 1, 1, 16)
    got = _stack(layers, x, _mask(kind, keep))
    assert torch.isfinite(got).all()
    assert torch.allclose(got[:, :n], _stack(layers, x[:, :n]), atol=1e-12)


@torch.no_grad()
def test_left_padding():
    layers, x, pad = _layers(2, window=5), _x(1, 14), 6
    got = _stack(layers, x, (torch.arange(14) >= pad)[None, None, None])
    assert torch.isfinite(got).all()
    # the rows of the padding see nothing, the gate's product with zeros is zero
    assert torch.equal(layers[0](x, attention_mask=(torch.arange(14) >= pad)[None, None, None]).output[:, :pad],
                       torch.zeros(1, pad, 64, dtype=torch.float64))


@torch.no_grad()
def test_weights_of_a_row_without_keys_are_zero():
    layer, x = _layers(1, window=3)[0], _x(1, 10)
    mask = (torch.arange(10) < 4)[None, None, None]
    w = layer(x, attention_mask=mask, output_attentions=True).attention_weights
    assert torch.equal(w[:, :, 6:], torch.zeros_like(w[:, :, 6:]))
    assert torch.allclose(w[:, :, :6].sum(-1), torch.ones(1, 4, 6, dtype=torch.float64))


@torch.no_grad()
def test_a_position_past_every_key():
    '''A tensor position (the exported step's) whose window starts behind the last key.'''
    layer, x = _layers(1, window=3)[0], _x(1, 2)
    assert torch.equal(layer(x, embedding_start=torch.tensor([9])).output, torch.zeros(1, 2, 64, dtype=torch.float64))


@pytest.mark.parametrize('kind', ['bool', 'additive'])
def test_gradients_stay_finite_and_are_the_valid_rows(kind):
    layers, n = _layers(2, window=3), 6
    keep = (torch.arange(12) < n)[None, None, None]
    grads = []
    for cut in (12, n):
        for layer in layers:
            layer.zero_grad()
        x = _x(1, 12)[:, :cut].requires_grad_()
        out = _stack(layers, x, _mask(kind, keep) if cut == 12 else None)
        out[:, :n].pow(2).sum().backward()
        grads.append([x.grad[:, :n]] + [p.grad for layer in layers for p in layer.parameters() if p.grad is not None])
        assert torch.isfinite(x.grad).all()
    assert len(grads[0]) == len(grads[1])
    for a, b in zip(*grads):
        assert torch.isfinite(a).all() and torch.allclose(a, b, atol=1e-10)
