'''One-launch Chord decode steps of many tokens (up to 16 query rows per kv head, so up to 16 new
positions where every query head has a kv head of its own): every new row reaches the cache, the
outputs are those of the several launches and of the formula in float64.'''
import pytest
import torch

from golden.weights import fill_params
from support import assert_bf16_close, gen
from window_ref import check_attention

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF = torch.bfloat16
# window, sinks; 61: new positions 64 - 3 .. behind the window's start, so that a step's rows lie in two
# tiles and two shares
WINDOWS = [(None, 0), (61, 0), (700, 3)]


def _layer(H, Hkv, window, sinks, seed=5):
    from motif.block.attention.chord_attn import ChordAttention
    layer = ChordAttention(hidden_size=64 * H, num_heads=H, num_kv_heads=Hkv, window=window, sinks=sinks)
    fill_params(layer, seed)
    return layer.to(DEV, BF).eval()


def _cache(B, Hkv, length, capacity, seed=11):
    '''Random rows up to `length`; what lies behind them is poisoned.'''
    from motif.model.cache import StaticKVLayerCache
    cache = StaticKVLayerCache().allocate(B, Hkv, capacity, 64, DEV, BF)
    rows = (0.5 * torch.randn(2, B, Hkv, length, 64, generator=gen(seed))).to(DEV, BF)
    for slab in cache._slab:
        slab.fill_(1000.)
    cache.fill(rows[0], rows[1])
    return cache


def _run(layer, cache, xs, fused):
    from motif.block.attention import chord_attn
    prev, chord_attn.FUSED_STEP = chord_attn.FUSED_STEP, fused
    try:
        return [layer(x, past_key_value=cache).output for x in xs]
    finally:
        chord_attn.FUSED_STEP = prev


@pytest.mark.parametrize('window,sinks', WINDOWS)
@pytest.mark.parametrize('B,H,Hkv,length,L', [(1, 2, 2, 120, 5), (2, 12, 12, 1000, 8), (3, 4, 4, 4090, 8), (1, 2, 2, 1, 7),
                                              (2, 4, 2, 250, 4)])
@torch.no_grad()
def test_layer_steps(B, H, Hkv, length, L, window, sinks):
    layer = _layer(H, Hkv, window, sinks)
    xs = [(0.5 * torch.randn(B, L, 64 * H, generator=gen(i))).to(DEV, BF) for i in range(3)]
    caches = [_cache(B, Hkv, length, length + 3 * L + 5) for _ in range(2)]
    got, ref = _run(layer, caches[0], xs, True), _run(layer, caches[1], xs, False)
    assert caches[0].step_workspace is not None and caches[1].step_workspace is None
    for cache in caches:
        assert cache.length == int(cache.length_dev) == length + 3 * L
    for a, b, what in zip(caches[0]._slab, caches[1]._slab, ('keys', 'values')):
        assert torch.equal(a, b), what
    for a, b in zip(got, ref):
        if window is None:
            assert torch.equal(a, b)
        else:  # (the sums run over other shares)
            assert_bf16_close(a, b)


@pytest.mark.parametrize('window,sinks', WINDOWS)
@pytest.mark.parametrize('H,Hkv,length,L', [(2, 2, 300, 16), (2, 2, 60, 9), (4, 2, 500, 8), (6, 2, 333, 5), (3, 3, 0, 13)])
@torch.no_grad()
def test_op_against_the_formula(H, Hkv, length, L, window, sinks):
    from motif.block.attention.chord_attn import LogPositions
    from motif.ops import chord_kv4_prep, kv4_alloc
    from motif.ops.chord_attention import chord_decode_step, chord_decode_step_serves, chord_decode_step_workspace
    B, cap = 2, length + 2 * L
    g = gen(H + L)
    par = (torch.exp(0.3 * torch.randn(H, generator=g)), 0.2 * torch.randn(H, generator=g), 0.2 * torch.randn(H, generator=g),
           1 + 0.1 * torch.randn(H, generator=g))
    qw, kw = ((1 + 0.1 * torch.randn(64, generator=g)).to(DEV, BF) for _ in range(2))
    cache = _cache(B, Hkv, length, cap)
    table = LogPositions.get(cap, torch.device(DEV, 0))
    work = chord_decode_step_workspace(B, H, Hkv, L, cap, torch.device(DEV, 0), window, sinks)
    for step in range(2):
        at = length + step * L
        proj = torch.randn(B, L, (H + 2 * Hkv) * 64, generator=g).to(DEV, BF)
        assert chord_decode_step_serves(proj, H, Hkv, 64)
        # (the step's query rows: the input kernel's, the same bits)
        q = chord_kv4_prep(proj, (0, 64 * H, 64 * (H + Hkv)), qw, kw, 1e-5, kv4_alloc(B, Hkv, cap, 64, DEV),
                           cache.length_dev, H).cpu()
        out = chord_decode_step(proj, (0, 64 * H, 64 * (H + Hkv)), qw, kw, 1e-5, *cache._slab, cache.length_dev,
                                *(t.to(DEV) for t in par), table, H, 0.125, 1e-5, work, window, sinks)
        assert int(cache.length_dev) == at + L
        heads = proj.cpu().view(B, L, H + 2 * Hkv, 64).transpose(1, 2)
        assert torch.equal(cache._slab[1][:, :, at:at + L].cpu(), heads[:, H + Hkv:]), 'values'
        x = heads[:, H:H + Hkv].double()
        k = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * kw.cpu().double()
        # two roundings to bf16, half a step (2^-8) each, and fp32's
        dk = (cache._slab[0][:, :, at:at + L].cpu().double() - k).abs()
        assert (dk <= (2 * 2.0 ** -8 + 2.0 ** -15) * k.abs()).all(), 'keys'
        log_n = torch.log(torch.arange(at + 1, at + L + 1, dtype=torch.float32))[None].expand(B, L)
        kk, vv = (s[:, :, :at + L].cpu() for s in cache._slab)
        check_attention(out, q, kk, vv, par, log_n, at, window, sinks, what=f'step {step}')
