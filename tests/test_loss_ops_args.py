'''What linear_cross_entropy, the row norms and dropout_add refuse, on the host, and their C
entries' checks (no kernel runs).'''
import ctypes

import pytest
import torch

from motif.ops import _lib, dropout_add, layer_norm_rows, linear_cross_entropy, rms_norm_rows

X, W, T = torch.zeros(6, 8), torch.zeros(10, 8), torch.zeros(6, dtype=torch.int64)


@pytest.mark.parametrize('args,kw,err', [
    ((X, W, T), dict(reduction='max'), ValueError),
    ((X, W[:, :7], T), {}, ValueError),
    ((X, W[0], T), {}, ValueError),
    ((X, W, T[:5]), {}, ValueError),
    ((X, W, T.float()), {}, ValueError),
    ((X, W[:0], T), {}, ValueError),
    ((X[:, :0], W[:, :0], T), {}, ValueError),
    ((X, W.bfloat16(), T), {}, ValueError),
    ((X.double(), W.double(), T), {}, NotImplementedError),
    ((X.half(), W.half(), T), {}, NotImplementedError),
    ((X[:1].expand(2 ** 23 + 1, 8), W, T[:1].expand(2 ** 23 + 1)), {}, ValueError),
    ((X, W[:1].expand(2 ** 22, 8), T), {}, ValueError),
    ((torch.zeros(1, 65537), torch.zeros(2, 65537), T[:1]), {}, ValueError),
    ((X, W, T), {}, ValueError),  # (not on a GPU)
])
def test_linear_cross_entropy(args, kw, err):
    with pytest.raises(err, match='linear_cross_entropy|unsupported dtype'):
        linear_cross_entropy(*args, **kw)


@pytest.mark.parametrize('fn', [rms_norm_rows, layer_norm_rows])
@pytest.mark.parametrize('x,w,err', [
    (X.double(), None, NotImplementedError),
    (X[:, :0], None, ValueError),
    (torch.tensor(1.0), None, ValueError),
    (torch.zeros(2, 16385), None, NotImplementedError),
    (X, W[0, :7], ValueError),
    (X, W[0].bfloat16(), ValueError),
    (X, W, ValueError),
    (X, W[0], ValueError),  # (not on a GPU)
])
def test_row_norms(fn, x, w, err):
    with pytest.raises(err, match=fn.__name__):
        fn(x, w)


def test_layer_norm_bias():
    with pytest.raises(ValueError, match='bias'):
        layer_norm_rows(X, W[0], W[0, :7])


@pytest.mark.parametrize('kw,err', [
    (dict(p=1.0), ValueError), (dict(p=-0.1), ValueError), (dict(p=float('nan')), ValueError),
    (dict(x=X.double()), NotImplementedError),
    (dict(residual=X[:5]), ValueError), (dict(residual=X[:1]), ValueError), (dict(residual=X.bfloat16()), ValueError),
    (dict(seed=2 ** 64), ValueError), (dict(seed=-2 ** 63 - 1), ValueError), (dict(seed=1.5), TypeError),
    (dict(seed=True), TypeError), (dict(seed=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(seed=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(), ValueError),  # (not on a GPU)
])
def test_dropout_add(kw, err):
    args = dict(x=X, p=0.5, seed=1)
    args.update(kw)
    with pytest.raises(err, match='dropout_add'):
        dropout_add(**args)


def _err():
    return _lib.lib().motif_last_error().decode()


def test_c_entries_check_their_arguments():
    lib = _lib.lib()
    P = ctypes.c_void_p(16)  # (never read: every call below ends at a check)
    big = 1 << 40

    def ce_fwd(x=P, N=6, d=8, V=10, red=2, rs=8, ws=P, nbytes=big, dtype=0):
        return lib.motif_linear_ce_fwd(x, rs, P, rs, P, 1, -100, N, d, V, red, P, P, P, ws, nbytes, dtype, None)
    for kw in (dict(x=None), dict(N=0), dict(d=0), dict(V=0), dict(N=2 ** 23 + 1), dict(V=2 ** 22), dict(d=65537, rs=65537), dict(red=3), dict(rs=7), dict(ws=None), dict(nbytes=16)):
        assert ce_fwd(**kw) == _lib.ERR_INVALID and 'linear_ce_fwd' in _err(), kw
    assert ce_fwd(dtype=2) == _lib.ERR_UNSUPPORTED

    def ce_bwd(w=P, N=6, d=8, V=10, red=2, rs=8, nbytes=big, dtype=0, dx=P, dw=P):
        return lib.motif_linear_ce_bwd(P, w, rs, P, P, 1, N, d, V, red, dx, dw, P, nbytes, dtype, None)
    for kw in (dict(w=None), dict(N=-1), dict(red=-1), dict(rs=7), dict(nbytes=16)):
        assert ce_bwd(**kw) == _lib.ERR_INVALID and 'linear_ce_bwd' in _err(), kw
    assert ce_bwd(dtype=2) == _lib.ERR_UNSUPPORTED
    assert ce_bwd(dx=None, dw=None) == 0

    def norm_bwd(dy=P, rows=4, D=8, mean=P, nbytes=big, layer=1, dtype=1, dx=P, dw=P):
        return lib.motif_row_norm_bwd(dy, 8, P, 8, P, P, mean, dx, 8, dw, None, rows, D, layer, P, nbytes, dtype, None)
    for kw in (dict(dy=None), dict(rows=0), dict(D=0), dict(mean=None), dict(nbytes=4)):
        assert norm_bwd(**kw) == _lib.ERR_INVALID and 'row_norm_bwd' in _err(), kw
    assert norm_bwd(D=16385) == _lib.ERR_UNSUPPORTED and norm_bwd(dtype=7) == _lib.ERR_UNSUPPORTED
    assert norm_bwd(dx=None, dw=None) == 0
    assert lib.motif_row_norm_fwd(P, 8, None, None, None, 8, None, None, 4, 8, 1e-5, 0, 1, None) == _lib.ERR_INVALID
    assert lib.motif_row_norm_fwd(P, 8, None, None, P, 8, P, None, 4, 8, 1e-5, 1, 1, None) == _lib.ERR_INVALID
    assert lib.motif_dropout_add(None, None, P, 4, 0, 1.0, 0, None, 0, None) == _lib.ERR_INVALID
    assert lib.motif_dropout_add(P, None, P, -1, 0, 1.0, 0, None, 0, None) == _lib.ERR_INVALID
    assert lib.motif_dropout_add(P, None, P, 4, 0, 1.0, 0, None, 9, None) == _lib.ERR_UNSUPPORTED
    assert lib.motif_dropout_add(None, None, None, 0, 0, 1.0, 0, None, 0, None) == 0


def test_workspace_sizes():
    lib = _lib.lib()
    assert lib.motif_linear_ce_rows_bytes(5, 100, 1) == 5 * 128 * 2
    assert lib.motif_linear_ce_rows_bytes(0, 100, 1) == 0 and lib.motif_linear_ce_workspace_bytes(5, 0, 16, 8, 3, 1, 0) == 0
    for N in (1, 300, 70000):
        for V in (1, 300, 50000):
            aligned, off = (lib.motif_linear_ce_workspace_bytes(N, 64, at, 64, V, 1, 1) for at in (16, 18))
            assert off >= aligned + V * 64 * 2 and aligned > lib.motif_linear_ce_rows_bytes(N, 64, 1)
            assert lib.motif_linear_ce_workspace_bytes(N, 64, 18, 64, V, 0, 1) >= N * 64 * 4
    assert lib.motif_row_norm_bwd_workspace_bytes(10, 64, 1) == 2 * 10 * 64 * 4
    assert lib.motif_row_norm_bwd_workspace_bytes(10 ** 6, 64, 0) <= 4096 * 64 * 4  # (no more rows than workgroups)


def test_model_options():
    import dataclasses

    from motif.model.config import MotifChordConfig
    from motif.model.motif import MotifChordModel
    cfg = MotifChordConfig(vocab_size=32, model_dim=64, num_heads=2, num_kv_heads=1, head_k_dim=32, block=('gdn', 'chord'), block_n=1)
    model = MotifChordModel(cfg)
    assert cfg.dropout == 0.0 and all(d.dropout == 0.0 for b in model.blocks for d in b.features)
    with pytest.raises(ValueError, match='fused_loss'):
        model(torch.zeros(1, 4, dtype=torch.int64), fused_loss=True)
    for p in (1.0, -0.5):
        with pytest.raises(ValueError, match='dropout'):
            MotifChordModel(dataclasses.replace(cfg, dropout=p))
    with pytest.raises(TypeError):
        MotifChordConfig(drop=0.1)


def test_dropout_survives_a_checkpoint(tmp_path):
    from motif.model.config import MotifChordConfig
    from motif.model.motif import MotifChordModel
    cfg = MotifChordConfig(vocab_size=32, model_dim=64, num_heads=2, num_kv_heads=1, head_k_dim=32, block=('gdn', 'chord'),
                           block_n=1, dropout=0.25)
    path = str(tmp_path / 'm.safetensors')
    MotifChordModel(cfg).save_pretrained(path)
    back = MotifChordModel.from_pretrained(path, verbose=False)
    assert back.config.dropout == 0.25 and back.blocks[0].features[1].dropout == 0.25
    assert MotifChordModel.from_pretrained(path, verbose=False, dropout=0.0).config.dropout == 0.0
