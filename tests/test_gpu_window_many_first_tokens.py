'''Gradients of windowed Chord attention where a large part of the keys are first tokens: few, long chunks of
the queries behind the windows.'''
import pytest
import torch

from support import gen
from test_gpu_chord_window_bwd import _grads, formula64
from window_ref import inputs, log_n_of

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.mark.parametrize('B,H,Hkv,L,S,q_start,window,sinks', [
    (1, 4, 2, 1500, 1500, 0, 40, 1400),
    (3, 12, 12, 900, 900, 0, 64, 800),      # (one chunk: 7 blocks of 36 heads pass 128)
    (2, 12, 3, 1300, 1300, 0, 30, 700),
    (1, 2, 1, 700, 1400, 700, 100, 1399),
])
def test_against_the_formula(B, H, Hkv, L, S, q_start, window, sinks):
    q, k, v, par = inputs(B, H, Hkv, L, S, 64, BF, seed=L)
    log_n = log_n_of(B, L, q_start)
    do = torch.randn(B, H, L, 64, generator=gen(1)).to(BF)
    want, lims = formula64(q, k, v, par, log_n, do, q_start, window, sinks)
    _, got = _grads(q, k, v, par, log_n, do, q_start, window, sinks)
    for name, g, w, lim in zip(('dq', 'dk', 'dv', 'dalpha', 'dbeta', 'dmu', 'dssmax'), got, want, lims):
        dist = (g.cpu().double() - w).abs()
        assert (dist <= lim).all(), f'{name}: worst {float((dist / lim).max()):.2f} of the limit'
