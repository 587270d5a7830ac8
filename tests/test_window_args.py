'''Refusals of the windowed and 4-bit operators, on the CPU.'''
import pytest
import torch

from motif.ops import KV4Slab, chord_attention_kv4, kv4_alloc, kv4_append, kv4_read
from motif.ops.chord_attention import apply_chord_attention, apply_chord_attention_varlen, check_window


@pytest.mark.parametrize('window,sinks', [(0, 0), (-1, 0), (1.5, 0), (True, 0), ('4', 0), (4, -1), (4, 1.0), (4, True),
                                          (None, 3)])
def test_bad_windows(window, sinks):
    with pytest.raises(ValueError):
        check_window(window, sinks)
    x = torch.zeros(1, 1, 4, 64)
    p = torch.zeros(1)
    for fn, extra in ((apply_chord_attention, ()), (apply_chord_attention_varlen, (torch.tensor([0, 4]),))):
        with pytest.raises(ValueError, match='window|sinks'):
            fn(x, x, x, p, p, p, p, torch.zeros(1, 4), *extra, window=window, sinks=sinks)


def test_good_windows():
    assert check_window(None, 0) == (None, 0)
    assert check_window(7, 3) == (7, 3)
    assert check_window(2 ** 40, 2 ** 40) == (2 ** 31 - 1, 2 ** 31 - 1)


def test_torch_form_of_a_row_that_sees_nothing():
    from motif.ops.autograd_path import chord_attention_torch
    g = torch.Generator().manual_seed(0)
    q = torch.randn(1, 2, 6, 16, generator=g, dtype=torch.float64, requires_grad=True)
    k, v = (torch.randn(1, 1, 3, 16, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    par = [torch.ones(2, dtype=torch.float64) for _ in range(4)]
    out = chord_attention_torch(q, k, v, *par, torch.ones(1, 6, dtype=torch.float64), 0, window=2)
    assert torch.equal(out[:, :, 4:], torch.zeros(1, 2, 2, 16, dtype=torch.float64))
    for t in torch.autograd.grad(out.sum(), (q, k, v)):
        assert torch.isfinite(t).all()


def _cpu_slab(B=1, Hkv=2, cap=8, D=64):
    return kv4_alloc(B, Hkv, cap, D, 'cpu')


def test_alloc():
    s = _cpu_slab()
    assert s.capacity == 8 and s.head_dim == 64 and s.k_params.shape == (1, 2, 8, 2, 2)
    assert kv4_alloc(1, 1, 4, 16, 'cpu').v_params.shape == (1, 1, 4, 1, 2)
    with pytest.raises(ValueError, match='head_dim'):
        kv4_alloc(1, 1, 4, 48, 'cpu')


def test_cpu_slabs_are_refused():
    s = _cpu_slab()
    rows = torch.zeros(1, 2, 1, 64)
    with pytest.raises(ValueError, match='CUDA'):
        kv4_append(s, rows, rows, 0)
    with pytest.raises(ValueError, match='CUDA'):
        kv4_read(s, 0, 1)
    p = torch.zeros(4)
    with pytest.raises(ValueError, match='CUDA'):
        chord_attention_kv4(torch.zeros(1, 4, 1, 64), s, p, p, p, p, torch.zeros(1, 1), 4)


def test_malformed_slabs_are_refused():
    s = _cpu_slab()
    rows = torch.zeros(1, 2, 1, 64)
    bad = [
        s._replace(k_codes=s.k_codes.to(torch.int16)),
        s._replace(v_codes=s.v_codes[:, :, :4]),
        s._replace(k_params=s.k_params.float()),
        s._replace(v_params=s.v_params[:, :, :, :1]),
        KV4Slab(*[t[:, :, :, :24] if t.dtype == torch.uint8 else t for t in s]),
        s._replace(k_codes=s.k_codes[0]),
    ]
    for b in bad:
        with pytest.raises(ValueError, match='kv4_append'):
            kv4_append(b, rows, rows, 0)


def test_gradients_are_refused():
    s = _cpu_slab()
    rows = torch.zeros(1, 2, 1, 64, requires_grad=True)
    with pytest.raises(RuntimeError, match='forward-only'):
        kv4_append(s, rows, rows, 0)
    p = torch.zeros(4)
    with pytest.raises(RuntimeError, match='forward-only'):
        chord_attention_kv4(torch.zeros(1, 4, 1, 64, requires_grad=True), s, p, p, p, p, torch.zeros(1, 1), 4)


def test_prep_into_a_slab_refuses_on_the_host():
    from motif.ops import chord_kv4_prep
    s, w = _cpu_slab(), torch.ones(64)
    with pytest.raises(ValueError, match='CUDA'):
        chord_kv4_prep(torch.zeros(1, 1, 512), (0, 256, 384), w, w, 1e-5, s, torch.zeros(1, dtype=torch.int32), 4)
