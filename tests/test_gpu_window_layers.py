'''The windowed Chord layer and the 4-bit cache on the model's own paths: prefill, later
pieces, decode at the device cursor (one launch and several), packed sequences, training,
and the captured decode step of a whole model.'''
import pytest
import torch

from golden.weights import fill_params
from support import assert_bf16_close, assert_fp32_close, gen
from window_ref import attention64, slab_values64

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF, F32 = torch.bfloat16, torch.float32


def _layer(dtype, H=4, Hkv=2, hidden=256, seed=3, **kw):
    from motif.block.attention.chord_attn import ChordAttention
    layer = ChordAttention(hidden_size=hidden, num_heads=H, num_kv_heads=Hkv, **kw)
    fill_params(layer, seed)
    return layer.to(DEV, dtype).eval()


def _x(B, L, dtype, dim=256, seed=0):
    return torch.randn(B, L, dim, generator=gen(seed)).to(dtype).to(DEV)


def _exact(layer, x):
    '''The layer in float64 on the CPU (its materialised path).'''
    import copy
    return copy.deepcopy(layer).cpu().double()(x.cpu().double()).output


def _model(dtype, seed=5, **kw):
    from motif.model.config import MotifChordConfig
    from motif.model.motif import MotifChordModel
    from motif.model.presets import init_random
    cfg = MotifChordConfig(vocab_size=160, model_dim=256, num_heads=4, num_kv_heads=2, head_k_dim=32,
                           block=('gdn', 'chord'), block_n=2, **kw)
    return init_random(MotifChordModel(cfg), std=0.05, seed=seed).to(DEV, dtype).eval()


@pytest.mark.parametrize('H,Hkv', [(4, 2), (4, 4), (4, 1)])
@torch.no_grad()
def test_layer_fp32_against_float64(H, Hkv):
    layer = _layer(F32, H, Hkv, window=37, sinks=3)
    x = _x(2, 150, F32)
    want = _exact(layer, x)
    assert_fp32_close(layer(x).output, want, 1e-4, 'prefill')
    cache = layer.cache_type()()
    parts = [layer(x[:, a:b], past_key_value=cache).output for a, b in ((0, 100), (100, 101), (101, 130), (130, 150))]
    assert_fp32_close(torch.cat(parts, 1), want, 1e-4, 'pieces over a growing cache')


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('fused', [True, False])
@torch.no_grad()
def test_cursor_decode_equals_prefill(dtype, fused, monkeypatch):
    from motif.block.attention import chord_attn
    from motif.model.cache import StaticKVLayerCache
    monkeypatch.setattr(chord_attn, 'FUSED_STEP', fused)
    layer = _layer(dtype, window=40, sinks=2)
    x = _x(2, 130, dtype)
    whole = layer(x).output
    cache = StaticKVLayerCache().allocate(2, 2, 140, 64, DEV, dtype)
    parts = [layer(x[:, :30], past_key_value=cache).output]
    parts += [layer(x[:, i:i + 1], past_key_value=cache).output for i in range(30, 128)]
    parts.append(layer(x[:, 128:130], past_key_value=cache).output)
    assert int(cache.length_dev) == cache.length == 130
    got = torch.cat(parts, 1)
    if dtype == F32:
        assert_fp32_close(got, whole, 1e-4)
    else:
        assert_bf16_close(got, whole)


@torch.no_grad()
def test_one_launch_step_against_several():
    '''The fused step and the input + decode kernels write the same rows; their sums run over
    other splits, so outputs agree to bf16 rounding.'''
    from motif.block.attention import chord_attn
    from motif.model.cache import StaticKVLayerCache
    outs, rows = [], []
    for fused in (True, False):
        chord_attn.FUSED_STEP = fused
        try:
            layer = _layer(BF, window=33, sinks=1)
            cache = StaticKVLayerCache().allocate(2, 2, 80, 64, DEV, BF)
            x = _x(2, 80, BF)
            layer(x[:, :20], past_key_value=cache)
            outs.append(torch.cat([layer(x[:, i:i + 1], past_key_value=cache).output for i in range(20, 80)], 1))
            rows.append(cache.k.clone())
        finally:
            chord_attn.FUSED_STEP = True
    assert torch.equal(rows[0], rows[1])
    assert_bf16_close(outs[0], outs[1])


@pytest.mark.parametrize('kind', ['rows', 'window', 'kv4'])
@torch.no_grad()
def test_steps_of_changing_lengths_over_one_cache(kind):
    '''Steps of 3, 1, 2 and 1 tokens: each has a scratch laid out for its own rows.'''
    from motif.model.cache import KV4LayerCache, StaticKVLayerCache
    layer = _layer(BF, **(dict(window=700, sinks=2) if kind == 'window' else {}))
    x = _x(1, 1510, BF)

    def run(steps):
        cache = (KV4LayerCache if kind == 'kv4' else StaticKVLayerCache)().allocate(1, 2, 1600, 64, DEV, BF)
        layer(x[:, :1500], past_key_value=cache)
        outs, at = [], 1500
        for n in steps:
            outs.append(layer(x[:, at:at + n], past_key_value=cache).output)
            at += n
        assert int(cache.length_dev) == cache.length == at
        return torch.cat(outs, 1)
    assert_bf16_close(run((3, 1, 2, 1, 3)), run((1,) * 10))


@torch.no_grad()
def test_masks_take_the_materialised_path_with_the_same_window():
    layer = _layer(F32, window=12, sinks=2)
    x = _x(2, 50, F32)
    got = layer(x, attention_mask=torch.ones(2, 50, dtype=torch.bool, device=DEV)[:, None, None]).output
    assert_fp32_close(got, layer(x).output, 1e-4)


@torch.no_grad()
def test_packed_sequences():
    layer = _layer(BF, window=20, sinks=2)
    lens = [33, 1, 70]
    x = _x(1, sum(lens), BF)
    cu = torch.tensor([0, 33, 34, 104], dtype=torch.int32, device=DEV)
    got = layer.forward_varlen(x, cu).output
    parts = [layer(x[:, a:b]).output for a, b in ((0, 33), (33, 34), (34, 104))]
    assert_bf16_close(got, torch.cat(parts, 1))


@torch.no_grad()
def test_kv4_layer_decodes_over_the_rows_as_held():
    from motif.model.cache import KV4LayerCache
    layer = _layer(F32, window=None)
    x = _x(2, 90, F32)
    cache = KV4LayerCache().allocate(2, 2, 96, 64, DEV, F32)
    first = layer(x[:, :70], past_key_value=cache).output
    assert_fp32_close(first, _exact(layer, x[:, :70]), 1e-4, 'a prompt attends to itself unrounded')
    for a, b in ((70, 71), (71, 73), (73, 90)):  # cursor steps, then a later piece
        got = layer(x[:, a:b], past_key_value=cache).output
        assert cache.length == int(cache.length_dev) == b
        k, v = (t[:, :, :b] for t in slab_values64(cache.slab))
        xs, n = x[:, a:b].cpu().double(), b - a
        l64 = __import__('copy').deepcopy(layer).cpu().double()
        q = l64.q_norm(l64.reshape_q(l64.q_proj(xs), n, 2))
        al, be, mu, ss = l64.ggd_params()
        ln = torch.log(torch.arange(a + 1, b + 1, dtype=torch.float64))[None].expand(2, n)
        out, _, _ = attention64(q, k, v, (al, be, mu, ss), ln, a)
        want = l64.o_proj(out.transpose(1, 2).reshape(2, n, 256)) * torch.sigmoid(l64.g_proj(xs))
        assert_fp32_close(got, want, 1e-4, f'rows {a}..{b}')
    kk, vv = cache.k, cache.v
    assert kk.shape == (2, 2, 90, 64) and torch.equal(kk.cpu(), slab_values64(cache.slab)[0][:, :, :90].float())
    assert torch.equal(vv.cpu(), slab_values64(cache.slab)[1][:, :, :90].float())


@pytest.mark.parametrize('kv_bits', [16, 4])
@pytest.mark.parametrize('kw', [dict(), dict(window=24, sinks=2)], ids=['all', 'window'])
@torch.no_grad()
def test_model_graph_replays_equal_eager_steps(kv_bits, kw):
    from motif.model.cache import ModelCache
    from motif.model.decode_graph import DecodeGraph
    model = _model(BF, **kw)
    ids = torch.randint(0, 160, (3, 80), generator=gen(2)).to(DEV)

    def prefilled():
        cache = ModelCache.for_decode(model, 3, 80, DEV, BF, kv_bits=kv_bits)
        model(ids[:, :50], cache=cache)
        return cache
    a, b = prefilled(), prefilled()
    graph = DecodeGraph(model, a, 3)
    for i in range(50, 80):
        got = graph.step(ids[:, i:i + 1]).clone()
        assert torch.equal(got, model(ids[:, i:i + 1], cache=b).logits), i
    for x, y in zip(a.layer_caches(), b.layer_caches()):
        assert x.length == y.length == 80
        if hasattr(x, 'length_dev'):
            assert int(x.length_dev) == 80
            for s, t in zip(x._slab, y._slab):
                assert torch.equal(s, t)
    with pytest.raises(RuntimeError, match='capacity'):
        graph.step(ids[:, :1])


@torch.no_grad()
def test_two_graphs_of_one_cache_and_a_reset():
    from motif.model.cache import ModelCache
    from motif.model.decode_graph import DecodeGraph
    model = _model(BF, window=24, sinks=2)
    ids = torch.randint(0, 160, (2, 64), generator=gen(2)).to(DEV)
    cache = ModelCache.for_decode(model, 2, 64, DEV, BF, kv_bits=4)
    runs = []
    graphs = [DecodeGraph(model, cache, 2), DecodeGraph(model, cache, 2)]
    for order in ((0, 0), (0, 1)):
        for lc in cache.layer_caches():
            lc.reset()
        for block in cache:
            block.attn_res.reset()
        model(ids[:, :40], cache=cache)
        runs.append(torch.cat([graphs[order[i % 2]].step(ids[:, i:i + 1]).clone() for i in range(40, 60)], 1))
    assert torch.equal(runs[0], runs[1])


@torch.no_grad()
def test_model_window_in_fp32_steps_equal_one_pass():
    from motif.model.cache import ModelCache
    model = _model(F32, window=16, sinks=1)
    ids = torch.randint(0, 160, (2, 60), generator=gen(3)).to(DEV)
    whole = model(ids).logits
    cache = ModelCache.for_decode(model, 2, 64, DEV, F32)
    parts = [model(ids[:, :40], cache=cache).logits] + [model(ids[:, i:i + 1], cache=cache).logits for i in range(40, 60)]
    assert_fp32_close(torch.cat(parts, 1), whole, 2e-4)
    wide = _model(F32, window=64)
    assert_fp32_close(wide(ids).logits, _model(F32)(ids).logits, 2e-4, 'a window of everything')


def test_model_trains_with_a_window():
    '''Gradients of a windowed bf16 model on the kernels against the same model's in fp32 (the
    torch form), as far apart as bf16 activations put them.'''
    ids = torch.randint(0, 160, (2, 96), generator=gen(4)).to(DEV)
    labels = torch.randint(0, 160, (2, 96), generator=gen(5)).to(DEV)
    grads = []
    for dtype in (BF, F32):
        model = _model(dtype, window=20, sinks=2).train()
        model(ids, labels=labels).loss.backward()
        grads.append({n: p.grad.float() for n, p in model.named_parameters() if p.grad is not None and 'chord' not in n})
    attn = [n for n in grads[0] if '.attn.' in n and ('theta_alpha' in n or 'ssmax' in n or 'q_proj' in n)]
    assert attn
    for n, g in grads[0].items():
        assert torch.isfinite(g).all(), n
    a = torch.cat([grads[0][n].flatten() for n in sorted(grads[0])])
    b = torch.cat([grads[1][n].flatten() for n in sorted(grads[0])])
    # two decoders deep, each bf16 tensor rounded to 2^-9 in the mean: a few per cent of the whole gradient
    assert float((a - b).norm() / b.norm()) < 0.1


@pytest.mark.parametrize('B,L,length,window,sinks', [(1, 1, 4200, 4000, 4), (2, 3, 2047, 1500, 40), (20, 2, 1200, 1000, 0),
                                                     (64, 1, 700, 600, 3), (1, 4, 60, 1, 0), (1, 1, 0, 5, 2)])
@torch.no_grad()
def test_one_launch_step_of_many_shares(B, L, length, window, sinks):
    '''From one to twelve workgroups a kv head: the rows and the cursor of the several launches, their output
    within bf16 rounding; three steps over one scratch, whose counters each leaves at zero.'''
    from motif.model.cache import StaticKVLayerCache
    from motif.block.attention import chord_attn
    layer = _layer(BF, window=window, sinks=sinks)
    rows = torch.randn(2, B, 2, length, 64, generator=gen(B), dtype=F32).to(DEV, BF)
    x = _x(B, 3 * L, BF)
    outs, slabs = [], []
    for fused in (True, False):
        chord_attn.FUSED_STEP = fused
        try:
            cache = StaticKVLayerCache().allocate(B, 2, length + 3 * L, 64, DEV, BF)
            cache.fill(rows[0], rows[1])
            outs.append(torch.cat([layer(x[:, L * i:L * i + L], past_key_value=cache).output for i in range(3)], 1))
        finally:
            chord_attn.FUSED_STEP = True
        assert cache.length == int(cache.length_dev) == length + 3 * L
        slabs.append(cache._slab)
    assert all(torch.equal(a, b) for a, b in zip(*slabs))
    assert_bf16_close(outs[0], outs[1])


@pytest.mark.parametrize('kind', ['rows', 'window', 'kv4'])
@torch.no_grad()
def test_a_step_of_another_length_captured_first(kind):
    '''A two-token step whose first run is a capture, after one-token steps: its replays, and eager steps
    of both lengths among them, equal eager steps throughout.'''
    from motif.model.cache import KV4LayerCache, StaticKVLayerCache
    layer = _layer(BF, **(dict(window=700, sinks=2) if kind == 'window' else {}))
    x = _x(2, 1420, BF)
    caches = [(KV4LayerCache if kind == 'kv4' else StaticKVLayerCache)().allocate(2, 2, 1500, 64, DEV, BF) for _ in range(2)]
    step = lambda cache, t: layer(t, past_key_value=cache).output
    for cache in caches:
        step(cache, x[:, :1400])
        step(cache, x[:, 1400:1401])
    buf, graph = x[:, :2].clone(), torch.cuda.CUDAGraph()
    length = caches[0].length
    with torch.cuda.graph(graph):
        got = step(caches[0], buf)
    caches[0].length = length
    at = 1401
    for n in (2, 2, 1, 2, -2, 1, 2):  # (-2: an eager step of two)
        part = x[:, at:at + abs(n)]
        if n == 2:
            buf.copy_(part)
            graph.replay()
            caches[0].advance(2)
            a = got
        else:
            a = step(caches[0], part)
        assert torch.equal(a, step(caches[1], part)), at
        at += abs(n)
    assert int(caches[0].length_dev) == int(caches[1].length_dev) == caches[0].length == at
