'''The scratch that a fixed-capacity cache keeps for its decode steps (a captured step holds its
address), on the CPU.'''
import pytest
import torch

from motif.model.cache import KV4LayerCache, StaticKVLayerCache

KINDS = [StaticKVLayerCache, KV4LayerCache]


def _cache(kind):
    return kind().allocate(1, 2, 8, 64, 'cpu', torch.bfloat16)


@pytest.mark.parametrize('kind', KINDS)
def test_a_move_that_moves_nothing_keeps_what_graphs_hold(kind):
    cache = _cache(kind)
    work = cache.workspace(('decode', 1, None, 0), lambda: torch.zeros(3))
    cache.log_table = table = torch.zeros(8)
    slab, cursor = tuple(cache._slab), cache.length_dev
    for kw in (dict(), dict(device='cpu'), dict(device=torch.device('cpu'), dtype=torch.bfloat16)):
        assert cache.to(**kw) is cache
        assert cache.workspace(('decode', 1, None, 0), lambda: torch.zeros(4)) is work
        assert cache.log_table is table and cache.length_dev is cursor
        assert all(a is b for a, b in zip(cache._slab, slab))


@pytest.mark.parametrize('kind', KINDS)
def test_a_move_leaves_nothing_of_the_old_place(kind):
    cache = _cache(kind)
    cache.workspace(('decode', 1, None, 0), lambda: torch.zeros(3))
    cache.log_table = torch.zeros(8)
    cache.to(device='meta')
    assert cache.decode_workspace is None and getattr(cache, 'log_table', None) is None
    assert all(t.device.type == 'meta' for t in (*cache._slab, cache.length_dev))


def test_another_dtype_of_the_rows_drops_the_scratch():
    cache = _cache(StaticKVLayerCache)
    cache.workspace(('decode', 1, None, 0), lambda: torch.zeros(3))
    assert cache.to(dtype=torch.float32).decode_workspace is None and cache.row_dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize('kv_bits', [16, 4])
@pytest.mark.parametrize('kw', [dict(), dict(window=600, sinks=2)], ids=['all', 'window'])
@torch.no_grad()
def test_replays_behind_a_move_that_moves_nothing(kv_bits, kw):
    from motif.model.cache import ModelCache
    from motif.model.config import MotifChordConfig
    from motif.model.decode_graph import DecodeGraph
    from motif.model.motif import MotifChordModel
    from motif.model.presets import init_random
    from support import gen
    cfg = MotifChordConfig(vocab_size=160, model_dim=256, num_heads=4, num_kv_heads=2, head_k_dim=32, block=('gdn', 'chord'),
                           block_n=1, **kw)
    model = init_random(MotifChordModel(cfg), std=0.05, seed=5).to('cuda', torch.bfloat16).eval()
    ids = torch.randint(0, 160, (1, 1510), generator=gen(2)).cuda()
    caches = [ModelCache.for_decode(model, 1, 1510, 'cuda', torch.bfloat16, kv_bits=kv_bits) for _ in range(2)]
    for cache in caches:
        model(ids[:, :1500], cache=cache)
    graph = DecodeGraph(model, caches[0], 1)
    for i in range(1500, 1506):
        for lc in caches[0].layer_caches():
            if isinstance(lc, StaticKVLayerCache):
                lc.to('cuda')
        junk = [torch.full((n,), float('nan'), device='cuda') for n in (64, 4096, 1 << 16, 1 << 18) for _ in range(8)]
        got = graph.step(ids[:, i:i + 1]).clone()
        assert torch.equal(got, model(ids[:, i:i + 1], cache=caches[1]).logits), i
        assert all(bool(t.isnan().all()) for t in junk)  # (nobody's scratch)
        del junk
