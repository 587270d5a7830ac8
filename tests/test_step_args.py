'''What chord_decode_step (the one-launch Chord step) refuses, on the host and before anything is launched.'''
import pytest
import torch

from motif.ops.chord_attention import chord_decode_step

B, H, HKV, L, CAP = 2, 4, 2, 1, 16
BF = torch.bfloat16


def _args(dev='cpu'):
    z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device=dev)
    return dict(proj=z(B, L, 64 * (H + 2 * HKV) + 64, dt=BF), offsets=(0, 64 * H, 64 * (H + HKV)),
                q_norm_weight=z(64, dt=BF), k_norm_weight=z(64, dt=BF), norm_eps=1e-5,
                k_cache=z(B, HKV, CAP, 64, dt=BF), v_cache=z(B, HKV, CAP, 64, dt=BF), length_dev=z(1, dt=torch.int32),
                alpha=z(H), beta=z(H), mu=z(H), ssmax=z(H), log_table=z(CAP), num_heads=H, softmax_scale=0.125, eps=1e-5,
                workspace=z(1 << 16, dt=torch.uint8))


def _wide(t):
    '''t's shape and values at a feature stride of 2.'''
    return torch.zeros(*t.shape, 2, dtype=t.dtype, device=t.device)[..., 0]


BAD = {
    'proj_dtype': (lambda a: dict(proj=a['proj'].float()), 'proj'),
    'proj_batch': (lambda a: dict(proj=a['proj'][:1]), 'proj'),
    'proj_stride': (lambda a: dict(proj=_wide(a['proj'])), 'proj'),
    'columns': (lambda a: dict(offsets=(0, 64 * H, 64 * (H + HKV) + 128)), 'columns'),
    'negative_column': (lambda a: dict(offsets=(-8, 64 * H, 64 * (H + HKV))), 'columns'),
    'heads': (lambda a: dict(num_heads=3), 'heads'),
    'rows': (lambda a: dict(proj=a['proj'].expand(B, 9, -1).contiguous()), '16 query rows'),
    'norm_shape': (lambda a: dict(q_norm_weight=a['q_norm_weight'][:32]), 'norm weights'),
    'norm_dtype': (lambda a: dict(k_norm_weight=a['k_norm_weight'].float()), 'norm weights'),
    'k_dtype': (lambda a: dict(k_cache=a['k_cache'].float()), 'caches'),
    'v_shape': (lambda a: dict(v_cache=a['v_cache'][:, :, :8]), 'caches'),
    'head_dim': (lambda a: dict(k_cache=a['k_cache'][..., :32], v_cache=a['v_cache'][..., :32]), 'caches'),
    'k_stride': (lambda a: dict(k_cache=_wide(a['k_cache'])), 'caches'),
    'length_dtype': (lambda a: dict(length_dev=a['length_dev'].long()), 'length_dev'),
    'no_length': (lambda a: dict(length_dev=a['length_dev'][:0]), 'length_dev'),
    'alpha_dtype': (lambda a: dict(alpha=a['alpha'].to(BF)), 'head parameters'),
    'mu_shape': (lambda a: dict(mu=a['mu'][:2]), 'head parameters'),
    'ssmax_stride': (lambda a: dict(ssmax=_wide(a['ssmax'])), 'head parameters'),
    'table_short': (lambda a: dict(log_table=a['log_table'][:8]), 'log_table'),
    'table_dtype': (lambda a: dict(log_table=a['log_table'].double()), 'log_table'),
    'workspace_dtype': (lambda a: dict(workspace=a['workspace'].float()), 'workspace'),
}
DEVICE = ['q_norm_weight', 'k_norm_weight', 'k_cache', 'v_cache', 'length_dev', 'alpha', 'beta', 'mu', 'ssmax', 'log_table',
          'workspace']


@pytest.mark.parametrize('window', [None, 8])
@pytest.mark.parametrize('name', BAD)
def test_refused_on_the_host(name, window):
    change, match = BAD[name]
    args = _args()
    args.update(change(args))
    with pytest.raises(ValueError, match=f'chord_decode_step: .*{match}'):
        chord_decode_step(**args, window=window)


@pytest.mark.parametrize('window', [None, 8])
@pytest.mark.parametrize('name', DEVICE)
def test_two_devices_are_refused(name, window):
    args = _args()
    args[name] = args[name].to('meta')
    with pytest.raises(ValueError, match='chord_decode_step: .*one device'):
        chord_decode_step(**args, window=window)


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(ValueError, match='CUDA'):
        chord_decode_step(**_args())


@pytest.mark.gpu
@pytest.mark.parametrize('window', [None, 8])
@torch.no_grad()
def test_refused_before_a_launch(window):
    args = _args('cuda')
    for change, match in BAD.values():
        with pytest.raises(ValueError, match=match):
            chord_decode_step(**{**args, **change(args)}, window=window)
    for name in DEVICE:
        with pytest.raises(ValueError, match='one device'):
            chord_decode_step(**{**args, name: args[name].cpu()}, window=window)
    assert int(args['length_dev']) == 0
    # and the same call as it should be
    assert torch.equal(chord_decode_step(**args, window=window).cpu(), torch.zeros(B, H, L, 64, dtype=BF))
    assert int(args['length_dev']) == 1
