'''What chord_decode_cursor refuses, on the host and before anything is launched.'''
import pytest
import torch

from motif.ops.chord_attention import chord_decode_cursor

B, H, HKV, L, CAP, D = 2, 4, 2, 1, 16, 64


def _args(dev='cpu'):
    z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device=dev)
    return dict(q=z(B, H, L, D), k_cache=z(B, HKV, CAP, D), v_cache=z(B, HKV, CAP, D),
                length_dev=z(1, dt=torch.int32), alpha=z(H), beta=z(H), mu=z(H), ssmax=z(H), log_table=z(CAP),
                log_n=z(B, L))


def _wide(t):
    '''t's shape and values at a feature stride of 2.'''
    return torch.zeros(*t.shape, 2, dtype=t.dtype, device=t.device)[..., 0]


BAD = [
    ('log_n', lambda a: dict(log_n=a['log_n'].to('meta')), 'log_n'),
    ('log_n_shape', lambda a: dict(log_n=a['log_n'][:1]), 'log_n'),
    ('log_n_dtype', lambda a: dict(log_n=a['log_n'].double()), 'log_n'),
    ('k_stride', lambda a: dict(k_cache=_wide(a['k_cache'])), 'feature stride'),
    ('v_stride', lambda a: dict(v_cache=_wide(a['v_cache'])), 'feature stride'),
    ('no_length', lambda a: dict(length_dev=a['length_dev'][:0]), 'length_dev'),
    ('workspace', lambda a: dict(workspace=torch.zeros(64, dtype=torch.uint8, device='meta')), 'workspace'),
]


@pytest.mark.parametrize('window', [None, 8])
@pytest.mark.parametrize('change,match', [b[1:] for b in BAD], ids=[b[0] for b in BAD])
def test_refused_on_the_host(change, match, window):
    args = _args()
    args.update(change(args))
    with pytest.raises(ValueError, match=match):
        chord_decode_cursor(**args, window=window)


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(ValueError, match='CUDA'):
        chord_decode_cursor(**_args(), window=8)


@pytest.mark.gpu
@pytest.mark.parametrize('window', [None, 8])
@torch.no_grad()
def test_refused_before_a_launch(window):
    args = _args('cuda')
    for change, match in (b[1:] for b in BAD[:6]):
        if match == 'log_n':
            bad = {**args, 'log_n': args['log_n'].cpu()}  # (a host pointer must not reach the kernel)
        else:
            bad = {**args, **change(args)}
        with pytest.raises(ValueError, match=match):
            chord_decode_cursor(**bad, window=window)
    assert int(args['length_dev']) == 0
    # and the same call as it should be
    assert torch.equal(chord_decode_cursor(**args, window=window).cpu(), torch.zeros(B, H, L, D))
    assert int(args['length_dev']) == 1
