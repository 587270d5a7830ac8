'''The 4-bit key / value cache: rows written and read back against the format's definition
(codes equal, values equal), attention over it against float64 of the values that the codes
stand for, refusals, cursor and captured forms.'''
import pytest
import torch

from support import gen
from window_ref import (check_attention, code_sizes64, inputs, log_n_of, over_rows64, quantise64, random_slab, slab_values64,
                        values64)

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = pytest.mark.parametrize('dtype', [BF, F16, F32], ids=['bf16', 'fp16', 'fp32'])


def _rows(B, Hkv, n, D, dtype, seed):
    g = gen(seed)
    k = torch.randn(B, Hkv, n, D, generator=g)
    v = 0.5 * torch.randn(B, Hkv, n, D, generator=g) + 2 * torch.randn(Hkv, 1, D, generator=g)
    k[:, :, ::3, ::5] *= 30     # outliers
    v[:, :, ::4] = 1.25         # constant rows
    v[:, :, 1::4, :16] = 0.0    # rows whose first features are zero
    return k.to(dtype), v.to(dtype)


@TYPES
@pytest.mark.parametrize('D', [16, 32, 64, 128])
@pytest.mark.parametrize('B,Hkv,cap,start,n', [(1, 1, 1, 0, 1), (2, 3, 40, 7, 1), (3, 2, 77, 5, 33), (1, 4, 300, 0, 300)])
@torch.no_grad()
def test_append_and_read(B, Hkv, cap, start, n, D, dtype):
    from motif.ops import kv4_append, kv4_read
    slab = random_slab(B, Hkv, cap, D, DEV, seed=D)
    before = [t.clone() for t in slab]
    k, v = _rows(B, Hkv, n, D, dtype, seed=n)
    kv4_append(slab, k.to(DEV), v.to(DEV), start)
    rows = slice(start, start + n)
    for name, x, codes, params, val in (('k', k, slab.k_codes, slab.k_params, 0), ('v', v, slab.v_codes, slab.v_params, 1)):
        code, scale, base = quantise64(x)
        c = codes[:, :, rows].cpu()
        assert torch.equal(torch.stack([c & 15, c >> 4], -1).flatten(-2), code.to(torch.uint8)), name
        assert torch.equal(params[:, :, rows].cpu(), torch.stack([scale, base], -1)), name
        want = values64(code, scale, base)
        for dt in (BF, F16, F32):
            got = kv4_read(slab, start, n, dt)[val].cpu()
            # the product is exact in fp32; one rounding there and one to dt
            assert torch.equal(got, want.float().to(dt)), (name, dt)
        # no value further off than half a step, the top of the range a rounding of scale and base more
        step = scale.double()[..., None].expand(*scale.shape, min(32, D)).flatten(-2)
        edge = 2.0 ** -8 * (x.double().abs().unflatten(-1, (-1, min(32, D))).amax(-1)[..., None] * 2
                            + 15 * scale.double()[..., None]).expand(*scale.shape, min(32, D)).flatten(-2)
        assert ((want - x.double()).abs() <= step / 2 + edge).all(), name
    for now, old in zip(slab, before):
        assert torch.equal(now[:, :, :start], old[:, :, :start]) and torch.equal(now[:, :, start + n:], old[:, :, start + n:])


@torch.no_grad()
def test_append_of_strided_rows_and_slab_views():
    from motif.ops import KV4Slab, kv4_append, kv4_read
    B, Hkv, n, D = 2, 3, 19, 64
    k, v = _rows(B, Hkv, n, D, BF, seed=4)
    base = random_slab(B + 2, Hkv + 1, 64, D, DEV, seed=1)
    slab = KV4Slab(*[t[1:1 + B, :Hkv, 8:40] for t in base])
    before = [t.clone() for t in base]
    kd = k.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    vd = torch.zeros(v.numel() + 1, dtype=BF, device=DEV)[1:].view(v.shape).copy_(v.to(DEV))
    kv4_append(slab, kd, vd, 3)
    got = kv4_read(slab, 3, n)
    for x, y in zip((k, v), got):
        assert torch.equal(y.cpu(), values64(*quantise64(x)).float().to(BF))
    for now, old in zip(base, before):
        mask = torch.ones(now.shape[:3], dtype=torch.bool, device=DEV)
        mask[1:1 + B, :Hkv, 11:11 + n] = False
        assert torch.equal(now[mask], old[mask])


@TYPES
@torch.no_grad()
def test_groups_that_are_not_finite_read_nan_and_no_other_does(dtype):
    from motif.ops import kv4_alloc, kv4_append, kv4_read
    k, v = _rows(1, 2, 6, 64, dtype, seed=2)
    k[0, 0, 1, 3] = float('nan')
    k[0, 1, 2, 40] = float('inf')
    v[0, 1, 5, 63] = -float('inf')
    slab = kv4_alloc(1, 2, 6, 64, DEV)
    kv4_append(slab, k.to(DEV), v.to(DEV), 0)
    for x, y in zip((k, v), kv4_read(slab, 0, 6, F32)):
        bad = ~torch.isfinite(x.float()).unflatten(-1, (-1, 32)).all(-1, keepdim=True).expand(1, 2, 6, 2, 32).flatten(-2)
        assert torch.equal(torch.isnan(y.cpu()), bad)


@torch.no_grad()
def test_largest_values_of_fp16_stay_finite():
    from motif.ops import kv4_alloc, kv4_append, kv4_read
    k = torch.full((1, 1, 1, 32), -65504.0, dtype=F16, device=DEV)
    v = torch.full((1, 1, 1, 32), 65504.0, dtype=F16, device=DEV)
    slab = kv4_alloc(1, 1, 1, 32, DEV)
    kv4_append(slab, k, v, 0)
    assert torch.equal(kv4_read(slab, 0, 1, F16)[0], k) and torch.equal(kv4_read(slab, 0, 1, F16)[1], v)


# B, H, Hkv, L, length, cap, D, window, sinks
SHAPES = [
    (1, 1, 1, 1, 1, 1, 64, None, 0),
    (1, 4, 1, 1, 31, 31, 64, None, 0),
    (2, 4, 2, 1, 65, 70, 64, None, 0),
    (1, 12, 3, 1, 300, 512, 64, None, 0),
    (3, 6, 2, 2, 129, 160, 64, None, 0),
    (1, 12, 3, 4, 517, 600, 64, None, 0),
    (2, 2, 2, 1, 700, 701, 64, 100, 3),
    (1, 12, 3, 1, 1000, 1001, 64, 333, 70),
    (1, 16, 1, 1, 400, 400, 64, 1, 0),
    (1, 16, 1, 3, 400, 400, 64, 1, 1),
    (2, 8, 2, 40, 200, 230, 64, None, 0),
    (1, 4, 2, 77, 77, 80, 64, 20, 2),
    (1, 4, 2, 1, 200, 200, 16, None, 0),
    (1, 4, 2, 3, 200, 200, 32, 50, 2),
    (2, 8, 2, 1, 333, 350, 128, None, 0),
    (1, 8, 2, 5, 333, 350, 128, 100, 40),
    (2, 4, 2, 0, 10, 16, 64, None, 0),
]


@TYPES
@pytest.mark.parametrize('shape', SHAPES, ids=[str(s) for s in SHAPES])
@torch.no_grad()
def test_attention(shape, dtype):
    from motif.ops import chord_attention_kv4
    B, H, Hkv, L, length, cap, D, window, sinks = shape
    slab = random_slab(B, Hkv, cap, D, DEV, seed=cap)
    q, _, _, par = inputs(B, H, Hkv, L, 1, D, dtype, seed=length)
    log_n = log_n_of(B, L, length - L)
    got = chord_attention_kv4(q.to(DEV), slab, *(t.to(DEV) for t in par), log_n.to(DEV), length, window=window, sinks=sinks)
    k, v = (t[:, :, :length] for t in slab_values64(slab))
    check_attention(got, q, k, v, par, log_n, length - L, window, sinks, what=str(shape),
                    rounded=code_sizes64(slab)[:, :, :length])


@TYPES
@pytest.mark.parametrize('window,sinks', [(None, 0), (60, 3)])
@torch.no_grad()
def test_rows_behind_the_length_and_outside_the_window_may_hold_anything(dtype, window, sinks):
    from motif.ops import chord_attention_kv4
    B, H, Hkv, L, length, cap = 2, 4, 2, 2, 333, 400
    slab = random_slab(B, Hkv, cap, 64, DEV, seed=3)
    q, _, _, par = inputs(B, H, Hkv, L, 1, 64, dtype, seed=1)
    args = [t.to(DEV) for t in (*par, log_n_of(B, L, length - L))]
    want = chord_attention_kv4(q.to(DEV), slab, *args, length, window=window, sinks=sinks)
    for t in (slab.k_params, slab.v_params):
        t[:, :, length:] = float('nan')
        if window:
            t[:, :, sinks:length - L - window + 1] = float('inf')
    got = chord_attention_kv4(q.to(DEV), slab, *args, length, window=window, sinks=sinks)
    assert torch.equal(got, want)


@TYPES
@pytest.mark.parametrize('window,sinks', [(None, 0), (37, 2)])
@pytest.mark.parametrize('D', [32, 64, 128])
@torch.no_grad()
def test_cursor_steps_equal_host_steps(dtype, window, sinks, D):
    from motif.ops import chord_attention_kv4, chord_decode_kv4_cursor, chord_decode_kv4_workspace, kv4_alloc, kv4_append
    B, H, Hkv, cap, L = 2, 6, 2, 130, 1
    table = torch.log(torch.arange(1, cap + 1, dtype=F32, device=DEV))
    slab = kv4_alloc(B, Hkv, cap, D, DEV)
    k, v = _rows(B, Hkv, cap, D, dtype, seed=D)
    k, v = k.to(DEV), v.to(DEV)
    first = 70
    kv4_append(slab, k[:, :, :first], v[:, :, :first], 0)
    _, _, _, par = inputs(B, H, Hkv, 1, 1, D, dtype, seed=2)
    par = [t.to(DEV) for t in par]
    cursor = torch.tensor([first], dtype=torch.int32, device=DEV)
    ws = chord_decode_kv4_workspace(B, H, Hkv, L, cap, D, dtype, DEV, window, sinks)
    pos = first
    while pos + L <= cap:
        q = inputs(B, H, Hkv, L, 1, D, dtype, seed=pos)[0].to(DEV)
        kv4_append(slab, k[:, :, pos:pos + L], v[:, :, pos:pos + L], cursor)
        got = chord_decode_kv4_cursor(q, slab, cursor, *par, table, window=window, sinks=sinks, workspace=ws)
        assert int(cursor) == pos + L
        kk, vv = (t[:, :, :pos + L] for t in slab_values64(slab))
        check_attention(got, q, kk, vv, par, table[None, pos:pos + L].expand(B, L), pos, window, sinks, what=f'pos {pos}',
                        rounded=code_sizes64(slab)[:, :, :pos + L])
        pos += L if pos < 75 else 9 if pos + 9 < cap else 1
        cursor.fill_(pos)
        kv4_append(slab, k[:, :, :min(pos, cap)], v[:, :, :min(pos, cap)], 0)


@torch.no_grad()
def test_append_past_the_capacity_is_dropped_on_the_device_and_refused_on_the_host():
    from motif.ops import kv4_alloc, kv4_append
    slab = kv4_alloc(1, 1, 4, 64, DEV)
    k, v = (t.to(DEV) for t in _rows(1, 1, 3, 64, BF, seed=1))
    for start in (-1, 2, 4):
        with pytest.raises(ValueError, match='outside'):
            kv4_append(slab, k, v, start)
    kv4_append(slab, k, v, torch.tensor([2], dtype=torch.int32, device=DEV))
    assert torch.equal(slab.k_codes[:, :, :2], torch.zeros_like(slab.k_codes[:, :, :2]))
    want = kv4_alloc(1, 1, 4, 64, DEV)
    kv4_append(want, k[:, :, :2], v[:, :, :2], 2)
    for a, b in zip(slab, want):
        assert torch.equal(a, b)


@torch.no_grad()
def test_refusals():
    from motif.ops import chord_attention_kv4, chord_decode_kv4_cursor, kv4_alloc, kv4_append, kv4_read
    slab = kv4_alloc(2, 2, 16, 64, DEV)
    p = torch.ones(4, device=DEV)
    q, ln = torch.zeros(2, 4, 1, 64, device=DEV, dtype=BF), torch.zeros(2, 1, device=DEV)
    ok = chord_attention_kv4(q, slab, p, p, p, p, ln, 16)
    assert torch.equal(ok, torch.zeros_like(ok))
    for bad in (dict(length=0), dict(length=17), dict(window=0), dict(sinks=2), dict(q=q[:, :3]), dict(q=q[:1]),
                dict(q=q.double()), dict(log_n=ln.double()), dict(log_n=ln[:1]), dict(alpha=p[:3]), dict(alpha=p.cpu()),
                dict(q=q.transpose(1, 3)), dict(out=torch.empty_like(q).float())):
        kw = dict(q=q, slab=slab, alpha=p, beta=p, mu=p, ssmax=p, log_n=ln, length=16)
        kw.update(bad)
        with pytest.raises(ValueError):
            chord_attention_kv4(**kw)
    rows = torch.zeros(2, 2, 1, 64, device=DEV)
    for k, v, s in ((rows, rows[:1], 0), (rows, rows.to(BF), 0), (rows[..., :32], rows[..., :32], 0), (rows, rows, 16),
                    (rows, rows, torch.zeros(1, device=DEV)), (rows, rows, torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            kv4_append(slab, k, v, s)
    for start, n in ((-1, 2), (0, 17), (3, -1)):
        with pytest.raises(ValueError):
            kv4_read(slab, start, n)
    with pytest.raises(NotImplementedError):
        kv4_read(slab, 0, 1, torch.float64)
    with pytest.raises(ValueError, match='back to back'):
        kv4_read(slab._replace(k_codes=slab.k_codes.expand(2, 2, 16, 32)[:, :, ::2], k_params=slab.k_params[:, :, ::2],
                               v_codes=slab.v_codes[:, :, ::2], v_params=slab.v_params[:, :, ::2]), 0, 1)
    cursor, table = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(16, device=DEV)
    for c, t in ((cursor.long(), table), (cursor.cpu(), table), (cursor, table[:15]), (cursor, table.double())):
        with pytest.raises(ValueError):
            chord_decode_kv4_cursor(q, slab, c, p, p, p, p, t)


@TYPES
@torch.no_grad()
def test_captured_steps_replay(dtype):
    '''Append and attention at the cursor in one graph; two graphs of the same cache.'''
    from motif.ops import chord_decode_kv4_cursor, kv4_alloc, kv4_append
    B, H, Hkv, cap, D = 2, 6, 2, 96, 64
    table = torch.log(torch.arange(1, cap + 1, dtype=F32, device=DEV))
    _, _, _, par = inputs(B, H, Hkv, 1, 1, D, dtype, seed=2)
    par = [t.to(DEV) for t in par]
    k, v = (t.to(DEV) for t in _rows(B, Hkv, cap, D, dtype, seed=8))
    qs = inputs(B, H, Hkv, cap, 1, D, dtype, seed=3)[0].to(DEV)
    eager, cur_e = kv4_alloc(B, Hkv, cap, D, DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    slab, cur = kv4_alloc(B, Hkv, cap, D, DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    q1, k1, v1 = qs[:, :, :1].clone(), k[:, :, :1].clone(), v[:, :, :1].clone()

    def step(s, c, q, kk, vv, window):
        kv4_append(s, kk, vv, c)
        return chord_decode_kv4_cursor(q, s, c, *par, table, window=window)
    graphs = []
    for window in (None, 20):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = step(slab, cur, q1, k1, v1, window)
        graphs.append((g, o, window))
    for i in range(40):
        g, o, window = graphs[i % 2]
        for dst, src in ((q1, qs), (k1, k), (v1, v)):
            dst.copy_(src[:, :, i:i + 1])
        g.replay()
        want = step(eager, cur_e, qs[:, :, i:i + 1], k[:, :, i:i + 1], v[:, :, i:i + 1], window)
        assert torch.equal(o, want), i
        if i % 8 == 0:
            torch.cuda.synchronize()
    assert int(cur) == int(cur_e) == 40
    for a, b in zip(slab, eager):
        assert torch.equal(a, b)


@pytest.mark.parametrize('dtype,D', [(BF, 16), (BF, 32), (BF, 64), (BF, 128), (F32, 16), (F32, 32), (F32, 64), (F32, 128)])
@pytest.mark.parametrize('B,L,H,Hkv,start', [(1, 1, 4, 1, 0), (3, 2, 6, 3, 17), (2, 5, 2, 2, 29)])
@torch.no_grad()
def test_prep_equals_norms_then_append(dtype, D, B, L, H, Hkv, start):
    '''The bits of the input kernel into plain rows followed by kv4_append; the last size's rows 32 .. pass
    the capacity and are dropped.'''
    from motif.block.attention.chord_attn import ChordAttention
    from motif.ops import chord_kv4_prep, kv4_alloc, kv4_append
    cap = 32
    layer = ChordAttention(hidden_size=H * D, num_heads=H, num_kv_heads=Hkv).to(DEV, dtype)
    g = torch.Generator().manual_seed(D + B)
    layer.q_norm.weight.copy_(1 + 0.2 * torch.randn(D, generator=g))
    layer.k_norm.weight.copy_(1 + 0.2 * torch.randn(D, generator=g))
    wide = torch.randn(B, L, (2 * H + 2 * Hkv) * D + 16, generator=g).to(DEV, dtype)
    wide[0, 0, H * D + 3] = float('inf') if B == 3 else 4.0
    proj = wide[..., :-16]
    ld = torch.tensor([start], dtype=torch.int32, device=DEV)
    slab, want = kv4_alloc(B, Hkv, cap, D, DEV), kv4_alloc(B, Hkv, cap, D, DEV)
    q = chord_kv4_prep(proj, (0, H * D, (H + Hkv) * D), layer.q_norm.weight, layer.k_norm.weight, layer.q_norm.eps,
                       slab, ld, H)
    qw = torch.empty_like(q)
    k, v = (torch.empty(B, Hkv, L, D, dtype=dtype, device=DEV) for _ in range(2))
    layer._prep(proj, qw, k, v, None, 0, L)
    kv4_append(want, k, v, ld)
    assert torch.equal(q, qw) and int(ld) == start
    for a, b in zip(slab, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@torch.no_grad()
def test_layer_of_head_dim_16_decodes():
    from motif.block.attention.chord_attn import ChordAttention
    from motif.model.cache import KV4LayerCache, StaticKVLayerCache
    torch.manual_seed(0)
    layer = ChordAttention(hidden_size=64, num_heads=4, num_kv_heads=2).to(DEV, BF).eval()
    x = torch.randn(2, 20, 64, generator=torch.Generator().manual_seed(1)).to(DEV, BF)
    for kind in (StaticKVLayerCache, KV4LayerCache):
        cache = kind().allocate(2, 2, 32, 16, DEV, BF)
        first = layer(x[:, :16], past_key_value=cache).output
        steps = [layer(x[:, i:i + 1], past_key_value=cache).output for i in range(16, 20)]
        assert int(cache.length_dev) == cache.length == 20
        whole = layer(x).output
        assert (first - whole[:, :16]).abs().max() < 2e-2
        if kind is StaticKVLayerCache:
            assert (torch.cat(steps, 1) - whole[:, 16:]).abs().max() < 2e-2


@torch.no_grad()
def test_prep_refusals():
    from motif.ops import chord_kv4_prep, kv4_alloc
    slab = kv4_alloc(2, 2, 16, 64, DEV)
    proj, w = torch.zeros(2, 1, 512, dtype=BF, device=DEV), torch.ones(64, dtype=BF, device=DEV)
    ld = torch.zeros(1, dtype=torch.int32, device=DEV)
    ok = dict(proj=proj, offsets=(0, 256, 384), q_norm_weight=w, k_norm_weight=w, norm_eps=1e-5, slab=slab, length_dev=ld,
              num_heads=4)
    assert chord_kv4_prep(**ok).shape == (2, 4, 1, 64)
    for bad in (dict(proj=proj[:1]), dict(proj=proj.half()), dict(proj=proj[0]), dict(offsets=(0, 256, 448)),
                dict(offsets=(0, 256)), dict(offsets=(-64, 256, 384)), dict(num_heads=3), dict(num_heads=10),
                dict(q_norm_weight=w[:32]), dict(k_norm_weight=w.float()), dict(length_dev=ld.long()),
                dict(length_dev=ld.cpu()), dict(length_dev=torch.zeros(2, dtype=torch.int32, device=DEV)),
                dict(proj=proj.transpose(0, 2).contiguous().transpose(0, 2))):
        with pytest.raises(ValueError, match='chord_kv4_prep'):
            chord_kv4_prep(**{**ok, **bad})
    odd = torch.zeros(2, 1, 516, dtype=BF, device=DEV)[..., 1:513]
    with pytest.raises(NotImplementedError, match='aligned'):
        chord_kv4_prep(**{**ok, 'proj': odd})


@pytest.mark.parametrize('dtype,L', [(BF, 1), (F16, 2), (BF, 70), (F32, 1)])
@torch.no_grad()
def test_long_cache_far_rows(dtype, L):
    '''Codes past 2^31 bytes from the start of the cache: written, read back and attended to.'''
    from motif.ops import chord_attention_kv4, kv4_alloc, kv4_append, kv4_read
    S, window, sinks = 70_000_000, 200, 3
    slab = kv4_alloc(1, 1, S, 64, DEV)  # 5.6 GB
    n = window + L
    far = [torch.randn(1, 1, n, 64, generator=gen(5 + i)).to(dtype).to(DEV) for i in range(2)]
    near = [torch.randn(1, 1, sinks, 64, generator=gen(7 + i)).to(dtype).to(DEV) for i in range(2)]
    kv4_append(slab, *far, S - n)
    kv4_append(slab, *near, torch.zeros(1, dtype=torch.int32, device=DEV))
    small = kv4_alloc(1, 1, n + sinks, 64, DEV)
    kv4_append(small, *(torch.cat([a, b], 2) for a, b in zip(near, far)), 0)
    for a, b in zip(kv4_read(slab, S - n, n, F32), kv4_read(small, sinks, n, F32)):
        assert torch.equal(a, b)
    q, _, _, par = inputs(1, 4, 1, L, 1, 64, dtype, seed=1)
    log_n = log_n_of(1, L, S - L)
    got = chord_attention_kv4(q.to(DEV), slab, *(t.to(DEV) for t in par), log_n.to(DEV), S, window=window, sinks=sinks)
    k, v = slab_values64(small)
    rows = list(range(sinks)) + list(range(S - n, S))
    want, mean = over_rows64(q, rows, k, v, par, log_n, S - L, window, sinks)
    # logits to 2^7 in fp32; 16-bit types: their weights' rounding (times codes to 15 steps) and the output's
    h = {BF: 2.0 ** -8, F16: 2.0 ** -11, F32: 0.0}[dtype]
    assert ((got.cpu().double() - want).abs() <= (2.0 ** -13 + 3 * h) * mean + h * want.abs()).all()
