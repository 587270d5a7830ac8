'''More rows than one launch of the norms' forward takes (2^32 threads, eight to a short row).'''
import pytest
import torch

from loss_ref import check, norm64

pytestmark = pytest.mark.gpu

DEV = 'cuda'
N = 2 ** 29 + 37
PLACES = (0, 2 ** 28, 2 ** 29 - 5000, N - 4096)  # (the second launch starts some 32 rows before 2^29)


@pytest.mark.parametrize('layer', [0, 1], ids=['rms', 'layer'])
def test_rows_of_one_feature(layer):
    from motif.ops import layer_norm_rows, rms_norm_rows
    g = torch.Generator(device=DEV).manual_seed(layer)
    x = torch.randn(N, 1, generator=g, device=DEV, dtype=torch.bfloat16).requires_grad_()
    dy = torch.randn(N, 1, generator=g, device=DEV, dtype=torch.bfloat16)
    w, b = (torch.tensor([v], device=DEV, dtype=torch.bfloat16) for v in (1.5, 0.25))
    y = layer_norm_rows(x, w, b, 0.1) if layer else rms_norm_rows(x, w, 0.1)
    dx, = torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        again = layer_norm_rows(x, w, b, 0.1) if layer else rms_norm_rows(x, w, 0.1)
    assert torch.equal(again, y)
    for at in PLACES:
        rows = slice(at, min(at + 10000, N))
        want = norm64(x[rows], w, b if layer else None, dy[rows], 0.1, layer)
        check(y[rows], *want[0], f'y from row {at}')
        check(dx[rows], *want[1], f'dx from row {at}')
