'''Windowed Chord attention with eps = 0: a key exactly mu positions away is at distance 0, where x^beta
is 0 and its derivative by beta is 0 as well (the limit of x^beta ln x).'''
import pytest
import torch

from window_ref import inputs, log_n_of

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF = torch.bfloat16


@pytest.mark.parametrize('mu', [0.0, -3.0])
@pytest.mark.parametrize('L,S,window,sinks', [(40, 40, 16, 0), (70, 200, 50, 3), (3, 3, 1, 0)])
def test_gradients_at_distance_zero(L, S, window, sinks, mu):
    from motif.ops import apply_chord_attention
    from motif.ops.autograd_path import chord_attention_torch
    B, H, Hkv = 2, 4, 2
    q, k, v, (al, _, _, ss) = inputs(B, H, Hkv, L, S, 64, BF, seed=L)
    par = (al, torch.tensor([1.0, 1.25, 1.5, 2.0]), torch.full((H,), mu), ss)
    log_n = log_n_of(B, L, S - L)
    do = torch.randn(B, H, L, 64, generator=torch.Generator().manual_seed(1)).to(BF)
    xs = [t.to(DEV).requires_grad_() for t in (q, k, v, *par)]
    out = apply_chord_attention(*xs, log_n.to(DEV), eps=0.0, window=window, sinks=sinks)
    got = torch.autograd.grad(out, xs, do.to(DEV))
    ys = [t.double().requires_grad_() for t in (q, k, v, *par)]
    ref = chord_attention_torch(*ys, log_n.double(), eps=0.0, window=window, sinks=sinks)
    want = torch.autograd.grad(ref, ys, do.double())
    with torch.no_grad():
        plain = apply_chord_attention(*xs, log_n.to(DEV), eps=0.0, window=window, sinks=sinks)
    for o in (out, plain):
        assert torch.isfinite(o).all()
        # a weight's and the output's rounding to bf16 (2^-8 each) of values up to the largest |v|
        assert float((o.detach().cpu().double() - ref.detach()).abs().max()) <= 2.0 ** -7 * float(v.abs().max()) + 1e-3
    for name, g, w in zip(('dq', 'dk', 'dv', 'dalpha', 'dbeta', 'dmu', 'dssmax'), got, want):
        g, w = g.cpu().double(), w.double()
        assert torch.isfinite(g).all(), name
        # bf16 gradients: P, dZ, O and the result rounded, 2^-8 of a term each, in the mean over a tensor
        assert float((g - w).norm()) <= 4 * 2.0 ** -8 * float(w.norm()) + 1e-3, name
