'''The window's place in the layers, the model and its checkpoints, and the 4-bit cache's
refusals, on the CPU (the Chord layer there computes with the materialised bias).'''
import json

import pytest
import torch

from motif.block.attention.chord_attn import ChordAttention
from motif.model.cache import KV4LayerCache, ModelCache
from motif.model.checkpoint import config_to_dict, load_checkpoint
from motif.model.config import MotifChordConfig
from motif.model.motif import MotifChordModel
from support import gen

CFG = dict(vocab_size=50, model_dim=64, num_heads=4, num_kv_heads=2, head_k_dim=16, block=('chord',), block_n=2)


def _x(B, L, dim=64, seed=0):
    return torch.randn(B, L, dim, generator=gen(seed), dtype=torch.float64)


def _layer(**kw):
    torch.manual_seed(0)
    layer = ChordAttention(hidden_size=64, num_heads=4, num_kv_heads=2, **kw).double().eval()
    with torch.no_grad():
        layer.theta_alpha.normal_(std=0.3)
        layer.theta_beta.normal_(std=0.2)
    return layer


@torch.no_grad()
def test_layer_sees_the_window_and_the_first_tokens_only():
    layer, x = _layer(window=5, sinks=2), _x(1, 20)
    base = layer(x).output
    for j in range(20):
        y = x.clone()
        y[:, j] += 1
        moved = ((layer(y).output - base).abs().amax(-1) > 0)[0]
        want = torch.tensor([j == i or (j < i and (i - j < 5 or j < 2)) for i in range(20)])
        assert torch.equal(moved, want), j


@torch.no_grad()
def test_layer_over_a_cache_equals_one_pass():
    layer, x = _layer(window=6, sinks=1), _x(2, 17)
    whole = layer(x).output
    cache = layer.cache_type()()
    parts = [layer(x[:, a:b], past_key_value=cache).output for a, b in ((0, 9), (9, 10), (10, 17))]
    assert torch.allclose(torch.cat(parts, 1), whole, atol=1e-12)


@torch.no_grad()
def test_no_window_is_the_default():
    a, b = _layer(), _layer(window=1000)
    assert a.window is None and a.sinks == 0
    assert torch.allclose(a(_x(1, 9)).output, b(_x(1, 9)).output, atol=1e-12)
    for bad in (dict(window=0), dict(sinks=3), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError):
            ChordAttention(hidden_size=64, num_heads=4, **bad)


def test_model_config_and_checkpoint(tmp_path):
    assert 'window' not in config_to_dict(MotifChordConfig(**CFG))
    cfg = MotifChordConfig(**CFG, window=7, sinks=2)
    assert {k: config_to_dict(cfg)[k] for k in ('window', 'sinks')} == {'window': 7, 'sinks': 2}
    model = MotifChordModel(cfg).eval()
    assert all(d.attn.window == 7 and d.attn.sinks == 2 for b in model.blocks for d in b.features)
    path = str(tmp_path / 'm.safetensors')
    model.save_pretrained(path)
    assert load_checkpoint(path).config == cfg
    back = MotifChordModel.from_pretrained(path, verbose=False)
    ids = torch.randint(0, 50, (1, 12), generator=gen(1))
    with torch.no_grad():
        want = model(ids).logits
        assert torch.equal(back(ids).logits, want)
        assert not torch.allclose(MotifChordModel.from_pretrained(path, verbose=False, window=2).eval()(ids).logits, want)
    json.dumps(config_to_dict(cfg))
    with pytest.raises(ValueError):
        MotifChordModel(MotifChordConfig(**CFG, sinks=2))


def test_kv4_cache_on_the_host():
    cache = KV4LayerCache().allocate(2, 2, 16, 64, 'cpu', torch.bfloat16)
    assert cache.capacity == 16 and cache.seq_length == 0 and cache.row_dtype == torch.bfloat16
    rows = torch.zeros(2, 2, 3, 64)
    with pytest.raises(ValueError, match='CUDA'):
        cache.update(rows, rows)
    with pytest.raises(TypeError):
        cache.append_slots(1, rows)
    with pytest.raises(TypeError):
        cache.adopt(rows, rows)
    cache.length = 15
    with pytest.raises(RuntimeError, match='capacity'):
        cache.update(rows, rows)
    cache.reset()
    assert cache.seq_length == 0 and int(cache.length_dev) == 0
    with pytest.raises(ValueError, match='grouped'):
        KV4LayerCache(num_heads=4)
    with pytest.raises(ValueError, match='head_dim'):
        KV4LayerCache().allocate(1, 1, 4, 48, 'cpu', torch.float32)
    model = MotifChordModel(MotifChordConfig(**CFG))
    with pytest.raises(ValueError, match='kv_bits'):
        ModelCache.for_decode(model, 1, 8, 'cpu', torch.float32, kv_bits=8)
    made = ModelCache.for_decode(model, 1, 8, 'cpu', torch.float32, kv_bits=4)
    assert all(type(c) is KV4LayerCache for c in made.layer_caches())
    plain = ModelCache.for_decode(model, 1, 8, 'cpu', torch.float32)
    assert not any(isinstance(c, KV4LayerCache) for c in plain.layer_caches())
    static = plain.layer_caches()
    for c in static:
        assert c.step_workspace is None and c.decode_workspace is None
        made = c.workspace(('decode', 1, None, 0), lambda: torch.zeros(3))
        assert c.decode_workspace is made and c.workspace(('decode', 1, None, 0), lambda: None) is made
        assert c.workspace(('decode', 2, None, 0), lambda: torch.zeros(4)).numel() == 4 and c.step_workspace is None
