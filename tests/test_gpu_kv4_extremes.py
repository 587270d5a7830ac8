'''4-bit rows of fp32 features near the largest number: bf16 ends at 3.3895e38, fp32 at 3.4028e38, and a
group whose smallest feature lies between them (below) still holds its finite features.'''
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = 'cuda'
F32 = torch.float32
BF_MAX = torch.finfo(torch.bfloat16).max


@pytest.mark.parametrize('D', [16, 32, 64, 128])
@torch.no_grad()
def test_groups_past_the_largest_bf16_number(D):
    from motif.ops import kv4_alloc, kv4_append, kv4_read
    big = 3.4e38
    rows = torch.zeros(1, 1, 4, D)
    rows[0, 0, 0] = torch.linspace(-big, -1.0, D)
    rows[0, 0, 1] = torch.linspace(1.0, big, D)
    rows[0, 0, 2] = -big
    rows[0, 0, 3] = big
    slab = kv4_alloc(1, 1, 4, D, DEV)
    kv4_append(slab, rows.to(DEV), (-rows).to(DEV), 0)
    for got, x in zip(kv4_read(slab, 0, 4, F32), (rows, -rows)):
        got, x = got.cpu().double(), x.double()
        assert torch.isfinite(got).all()
        grp = x.unflatten(-1, (-1, min(32, D)))
        step = (grp.amax(-1, keepdim=True) - grp.amin(-1, keepdim=True)) / 15
        # half a step, scale's rounding (2^-8 of it, 15 times), base's (2^-8 of the smallest feature) and, where the
        # base is held at the largest bf16 number, what lies between (4e-3 of it)
        lim = step * (0.5 + 15 * 2.0 ** -8) + (2.0 ** -8 + 4e-3) * grp.amin(-1, keepdim=True).abs() + 2.0 ** -20 * grp.abs()
        assert ((got.unflatten(-1, (-1, min(32, D))) - grp).abs() <= lim).all()


@torch.no_grad()
def test_the_input_kernel_writes_the_same():
    '''chord_kv4_prep's value rows (fp32) go through the same codes.'''
    from motif.ops import chord_kv4_prep, kv4_alloc, kv4_append
    g = torch.Generator().manual_seed(0)
    proj = torch.randn(2, 3, 4 * 64, generator=g)
    proj[:, 0, 192:] = torch.linspace(-3.4e38, -1.0, 64)
    proj[1, 1, 192:] = 3.4e38
    proj = proj.to(DEV)
    a, b = kv4_alloc(2, 1, 4, 64, DEV), kv4_alloc(2, 1, 4, 64, DEV)
    w = torch.ones(64, device=DEV)
    chord_kv4_prep(proj, (0, 128, 192), w, w, 1e-5, a, torch.zeros(1, dtype=torch.int32, device=DEV), 2)
    v = proj[:, None, :, 192:].contiguous()
    kv4_append(b, v, v, 0)
    assert torch.equal(a.v_codes, b.v_codes) and torch.equal(a.v_params, b.v_params)
    assert torch.isfinite(a.v_params.float()).all()
