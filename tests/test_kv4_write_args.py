'''4-bit rows are never written into a slab whose batch rows or heads share memory: every one of them would
write the same bytes, in no order.'''
import pytest
import torch

from motif.ops import KV4Slab, chord_kv4_prep, kv4_alloc, kv4_append, kv4_read


def _expanded(dim, dev='cpu'):
    one = kv4_alloc(1 if dim == 0 else 2, 1 if dim == 1 else 3, 8, 64, dev)
    return KV4Slab(*[t.expand(2, 3, *t.shape[2:]) for t in one])


@pytest.mark.parametrize('dim', [0, 1])
@pytest.mark.parametrize('which', range(4))
def test_writes_into_expanded_slabs_are_refused(dim, which):
    whole, shared = kv4_alloc(2, 3, 8, 64, 'cpu'), _expanded(dim)
    slab = KV4Slab(*[shared[i] if i == which else whole[i] for i in range(4)])
    rows = torch.zeros(2, 3, 1, 64)
    with pytest.raises(ValueError, match='kv4_append: .*share memory'):
        kv4_append(slab, rows, rows, 0)
    w = torch.ones(64)
    with pytest.raises(ValueError, match='chord_kv4_prep: .*share memory'):
        chord_kv4_prep(torch.zeros(2, 1, 64 * 9), (0, 192, 384), w, w, 1e-5, slab, torch.zeros(1, dtype=torch.int32), 3)


def test_single_rows_of_any_stride_are_not_taken_for_shared():
    '''(a batch or head of one: its stride is not used)'''
    slab = KV4Slab(*[t.as_strided(t.shape, (0, 0, *t.stride()[2:])) for t in kv4_alloc(1, 1, 8, 64, 'cpu')])
    rows = torch.zeros(1, 1, 1, 64)
    with pytest.raises(ValueError, match='CUDA'):
        kv4_append(slab, rows, rows, 0)


@pytest.mark.gpu
@torch.no_grad()
def test_expanded_slabs_are_read_and_single_rows_written():
    from motif.ops import chord_attention_kv4
    g = torch.Generator().manual_seed(0)
    rows = torch.randn(1, 1, 8, 64, generator=g).cuda()
    one = KV4Slab(*[t.as_strided(t.shape, (0, 0, *t.stride()[2:])) for t in kv4_alloc(1, 1, 8, 64, 'cuda')])
    kv4_append(one, rows, -rows, 0)
    shared = KV4Slab(*[t.expand(2, 3, *t.shape[2:]) for t in one])
    k, v = kv4_read(shared, 0, 8, torch.float32)
    whole = kv4_alloc(2, 3, 8, 64, 'cuda')
    kv4_append(whole, rows.expand(2, 3, 8, 64), -rows.expand(2, 3, 8, 64), 0)
    for a, b in zip((k, v), kv4_read(whole, 0, 8, torch.float32)):
        assert torch.equal(a, b)
    q, par = torch.randn(2, 6, 2, 64, generator=g).bfloat16().cuda(), [torch.ones(6, device='cuda') for _ in range(4)]
    log_n = torch.ones(2, 2, device='cuda')
    assert torch.equal(chord_attention_kv4(q, shared, *par, log_n, 8), chord_attention_kv4(q, whole, *par, log_n, 8))
