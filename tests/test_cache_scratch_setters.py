'''A caller's own scratch for the decode steps of a fixed-capacity cache: set as an attribute, used by the next
step of its kind, or dropped with None (CPU).'''
import pytest
import torch

from motif.model.cache import KV4LayerCache, StaticKVLayerCache


@pytest.mark.parametrize('kind', [StaticKVLayerCache, KV4LayerCache])
@pytest.mark.parametrize('name', ['decode', 'step'])
def test_set_used_and_dropped(kind, name):
    cache = kind().allocate(1, 2, 8, 64, 'cpu', torch.bfloat16)
    attr = f'{name}_workspace'
    other = 'step_workspace' if name == 'decode' else 'decode_workspace'
    mine, made = torch.zeros(16, dtype=torch.uint8), torch.zeros(8)
    assert getattr(cache, attr) is None
    setattr(cache, attr, mine)
    assert getattr(cache, attr) is mine and getattr(cache, other) is None
    assert cache.workspace((name, 1, None, 0), lambda: made) is mine
    # a step of another length lays its scratch out its own way
    assert cache.workspace((name, 2, None, 0), lambda: made) is made
    assert cache.workspace((name, 1, None, 0), lambda: made) is mine and getattr(cache, attr) is mine
    setattr(cache, attr, None)
    assert getattr(cache, attr) is None
    assert cache.workspace((name, 2, None, 0), lambda: mine) is mine
    # another one replaces all of the kind
    again = torch.zeros(16, dtype=torch.uint8)
    setattr(cache, attr, again)
    assert getattr(cache, attr) is again and cache.workspace((name, 2, None, 0), lambda: made) is again


def test_one_kind_leaves_the_other():
    cache = StaticKVLayerCache().allocate(1, 2, 8, 64, 'cpu', torch.bfloat16)
    step = cache.workspace(('step', 1, None, 0), lambda: torch.zeros(3))
    cache.decode_workspace = None
    assert cache.step_workspace is step
    cache.decode_workspace = torch.zeros(4)
    cache.allocate(1, 2, 8, 64, 'cpu', torch.bfloat16)
    assert cache.decode_workspace is None and cache.step_workspace is None


@pytest.mark.gpu
@pytest.mark.parametrize('window', [None, 600])
@torch.no_grad()
def test_layer_steps_over_the_callers_scratch(window):
    from golden.weights import fill_params
    from motif.block.attention import chord_attn
    from motif.ops.chord_attention import chord_decode_step_workspace
    from support import gen
    layer = chord_attn.ChordAttention(hidden_size=256, num_heads=4, num_kv_heads=2, window=window)
    fill_params(layer, 3)
    layer = layer.to('cuda', torch.bfloat16).eval()
    rows = torch.randn(2, 2, 2, 1500, 64, generator=gen(1)).to('cuda', torch.bfloat16)
    xs = [torch.randn(2, 1, 256, generator=gen(i)).to('cuda', torch.bfloat16) for i in range(3)]
    outs = []
    for own in (True, False):
        cache = StaticKVLayerCache().allocate(2, 2, 1510, 64, 'cuda', torch.bfloat16)
        cache.fill(*rows)
        if own:
            cache.step_workspace = mine = chord_decode_step_workspace(2, 4, 2, 1, 1510, rows.device, window)
            mine[:-20] = 255  # (all but the arrival counters of 2 x 2 kv heads)
        outs.append([layer(x, past_key_value=cache).output for x in xs])
        if own:
            assert cache.step_workspace is mine and not bool((mine[:64] == 255).all())
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    # too small a scratch is refused by the step that would use it
    cache = StaticKVLayerCache().allocate(2, 2, 1510, 64, 'cuda', torch.bfloat16)
    cache.fill(*rows)
    cache.step_workspace = torch.zeros(16, dtype=torch.uint8, device='cuda')
    with pytest.raises(ValueError, match='workspace too small'):
        layer(xs[0], past_key_value=cache)
