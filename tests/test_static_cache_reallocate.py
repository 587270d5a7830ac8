'''allocate() on a cache that was in use starts anew: nothing of the old place is left (CPU).'''
import pytest
import torch

from motif.model.cache import KV4LayerCache, StaticKVLayerCache


@pytest.mark.parametrize('kind', [StaticKVLayerCache, KV4LayerCache])
def test_nothing_of_the_old_place(kind):
    cache = kind().allocate(1, 2, 8, 64, 'cpu', torch.bfloat16)
    cache.workspace(('decode', 1, None, 0), lambda: torch.zeros(3))
    cache.log_table = torch.zeros(8)
    cache.length = 5
    cache.allocate(2, 2, 8, 64, 'meta', torch.bfloat16)
    assert getattr(cache, 'log_table', None) is None and cache.decode_workspace is None and cache.length == 0
    assert all(t.device.type == 'meta' and t.shape[0] == 2 for t in cache._slab) and cache.length_dev.device.type == 'meta'
