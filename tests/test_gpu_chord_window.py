'''Chord attention under a sliding window with visible first tokens, against float64: sizes,
types and head dims at the edges (rows that see nothing, windows of one key, first tokens
inside, beside and past the window), strides, rows that no query sees, the cursor form.'''
import pytest
import torch

from support import gen
from window_ref import attention64, check_attention, inputs, log_n_of, over_rows64

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _run(q, k, v, par, log_n, **kw):
    from motif.ops import apply_chord_attention
    return apply_chord_attention(*(t.to(DEV) for t in (q, k, v, *par, log_n)), **kw)


# B, H, Hkv, L, S, q_start, D, window, sinks
SHAPES = [
    (1, 1, 1, 1, 1, 0, 64, 1, 0),          # one token
    (1, 2, 1, 1, 200, 199, 64, 1, 0),      # a window of the query's own key
    (2, 4, 2, 1, 300, 299, 64, 64, 4),     # a decode row, first tokens apart from the window
    (1, 12, 3, 2, 517, 515, 64, 130, 1),
    (3, 4, 1, 4, 100, 96, 64, 33, 40),     # first tokens past the window's start
    (2, 4, 4, 33, 33, 0, 64, 16, 0),
    (1, 8, 2, 100, 100, 0, 64, 1, 1),
    (1, 4, 2, 257, 257, 0, 64, 100, 3),
    (2, 6, 2, 130, 400, 270, 64, 65, 33),  # a later piece
    (1, 4, 1, 65, 300, 235, 64, 31, 0),
    (1, 3, 3, 300, 300, 0, 64, 1000, 0),   # a window wider than the context
    (1, 4, 2, 70, 70, 0, 64, 8, 500),      # every token a first token
    (1, 2, 1, 200, 64, 0, 64, 20, 0),      # queries past the keys: rows that see nothing
    (1, 4, 4, 40, 16, 100, 64, 16, 0),     # every row sees nothing
    (1, 4, 4, 40, 16, 100, 64, 16, 2),     # every row sees the first tokens only
    (1, 4, 2, 150, 150, 0, 16, 40, 2),
    (1, 4, 2, 150, 150, 0, 32, 40, 2),
    (1, 4, 2, 150, 150, 0, 128, 40, 2),
    (1, 4, 2, 60, 150, 90, 24, 40, 2),     # head dims between the kernels'
    (1, 2, 2, 3, 90, 87, 80, 17, 5),
    (1, 4, 2, 500, 500, 0, 64, 450, 3),    # long windows of few blocks
    (2, 4, 1, 130, 700, 570, 64, 400, 20),
    (1, 3, 3, 433, 600, 167, 64, 600, 0),
    (1, 4, 4, 60, 500, 480, 64, 900, 1),   # queries past the keys
    (1, 8, 2, 90, 450, 700, 64, 380, 0),   # the last of them see nothing
    (3, 12, 3, 250, 250, 0, 64, 70, 2),    # more blocks than CUs
    (3, 12, 3, 250, 1100, 850, 64, 1000, 2),
    (1, 2, 1, 40, 1000, 960, 64, 900, 0),  # one short block under a long window
]


@pytest.mark.parametrize('dtype', [BF, F16, F32], ids=['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('shape', SHAPES, ids=[str(s) for s in SHAPES])
@torch.no_grad()
def test_forward(shape, dtype):
    B, H, Hkv, L, S, q_start, D, window, sinks = shape
    q, k, v, par = inputs(B, H, Hkv, L, S, D, dtype, seed=sum(shape))
    log_n = log_n_of(B, L, q_start)
    got = _run(q, k, v, par, log_n, q_start=q_start, window=window, sinks=sinks)
    assert got.dtype == dtype and got.shape == (B, H, L, D)
    check_attention(got, q, k, v, par, log_n, q_start, window, sinks, what=str(shape))


@pytest.mark.parametrize('dtype', [BF, F16, F32], ids=['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('L', [1, 4, 70])
@torch.no_grad()
def test_rows_that_no_query_sees_may_hold_anything(dtype, L):
    S, window, sinks = 333, 50, 3
    q, k, v, par = inputs(2, 4, 2, L, S, 64, dtype, seed=L)
    log_n = log_n_of(2, L, S - L)
    want = _run(q, k, v, par, log_n, window=window, sinks=sinks)
    for bad in (float('nan'), float('inf'), -float('inf')):
        k2, v2 = k.clone(), v.clone()
        k2[:, :, sinks:S - L - window + 1] = bad
        v2[:, :, sinks:S - L - window + 1] = bad
        assert torch.equal(_run(q, k2, v2, par, log_n, window=window, sinks=sinks), want)


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
@torch.no_grad()
def test_strides_and_destinations(dtype):
    from motif.ops import apply_chord_attention
    B, H, Hkv, L, S, D, window, sinks = 2, 4, 2, 90, 140, 64, 37, 2
    q, k, v, par = inputs(B, H, Hkv, L, S, D, dtype, seed=5)
    log_n = log_n_of(B, L, S - L)
    want = _run(q, k, v, par, log_n, window=window, sinks=sinks)
    args = [t.to(DEV) for t in (*par, log_n)]
    # [B, L, H, D] storage, rows inside wider ones, an odd start, one batch row for all
    qt = q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.zeros(B, S, Hkv * D + 8, dtype=dtype, device=DEV)
    wide[..., 8:] = k.to(DEV).transpose(1, 2).reshape(B, S, Hkv * D)
    kt = wide[..., 8:].view(B, S, Hkv, D).transpose(1, 2)
    odd = torch.zeros(v.numel() + 1, dtype=dtype, device=DEV)[1:].view(v.shape).copy_(v.to(DEV))
    out = torch.full((B, L, H, D), 7.0, dtype=dtype, device=DEV)
    got = apply_chord_attention(qt, kt, odd, *args, window=window, sinks=sinks, out=out.transpose(1, 2))
    assert torch.equal(got, want) and got.data_ptr() == out.data_ptr()
    one = apply_chord_attention(qt[:1].expand(B, H, L, D), kt[:1].expand(B, Hkv, S, D), odd[:1].expand(B, Hkv, S, D),
                                *args, window=window, sinks=sinks)
    assert torch.equal(one[0], want[0]) and torch.equal(one[1], want[0])
    flip = apply_chord_attention(qt, kt.flip(2).flip(2), v.to(DEV), *args, window=window, sinks=sinks)
    assert torch.equal(flip, want)


@pytest.mark.parametrize('dtype', [BF, F16], ids=['bf16', 'fp16'])
@torch.no_grad()
def test_packed_equals_sequences_apart(dtype):
    from motif.ops import apply_chord_attention, apply_chord_attention_varlen
    lens = [1, 70, 0, 133, 64, 5]
    T = sum(lens)
    q, k, v, par = inputs(1, 4, 2, T, T, 64, dtype, seed=9)
    log_n = torch.cat([log_n_of(1, n, 0) for n in lens], 1)
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)
    args = [t.to(DEV) for t in (q, k, v, *par, log_n)]
    got = apply_chord_attention_varlen(*args, cu.to(DEV), window=40, sinks=2)
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        if b > a:
            one = apply_chord_attention(*(t[:, :, a:b] for t in args[:3]), *args[3:7], args[7][:, a:b], window=40, sinks=2)
            if dtype == F16 or b - a > 8:  # (short bf16 sequences on their own are decodes)
                assert torch.equal(got[:, :, a:b], one)
            check_attention(got[:, :, a:b].cpu(), *(t[:, :, a:b] for t in (q, k, v)), par, log_n[:, a:b], 0, 40, 2, what=str((a, b)))


@pytest.mark.parametrize('H,Hkv', [(2, 2), (4, 2), (8, 2)])
@torch.no_grad()
def test_packed_sequences_see_themselves_only(H, Hkv):
    from motif.ops import apply_chord_attention_varlen
    from motif.ops.packed import PackedSeqs
    lens = [3, 17, 1, 0, 200, 64, 129, 2, 0]
    T = sum(lens)
    q, k, v, par = inputs(1, H, Hkv, T, T, 64, BF, seed=H)
    log_n = torch.cat([log_n_of(1, n, 0) for n in lens], 1)
    ps = PackedSeqs(torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()]))  # (boundaries on the host)
    run = lambda k, v: apply_chord_attention_varlen(*(t.to(DEV) for t in (q, k, v, *par, log_n)), ps, window=30, sinks=2)
    got = run(k, v)
    for a, b in ps.bounds():
        if b > a:
            check_attention(got[:, :, a:b].cpu(), *(t[:, :, a:b] for t in (q, k, v)), par, log_n[:, a:b], 0, 30, 2)
    for a, b in ps.bounds():  # rows of one sequence are nothing to the others
        if b > a:
            k2, v2 = k.clone(), v.clone()
            k2[:, :, a:b] = v2[:, :, a:b] = float('nan')
            other = run(k2, v2)
            assert torch.equal(other[:, :, :a], got[:, :, :a]) and torch.equal(other[:, :, b:], got[:, :, b:])


@torch.no_grad()
def test_packed_call_replays():
    from motif.ops import apply_chord_attention_varlen
    from motif.ops.packed import PackedSeqs
    ps = PackedSeqs(torch.tensor([0, 40, 41, 170]), 170, torch.device(DEV, 0))
    q, k, v, par = (inputs(1, 4, 2, 170, 170, 64, BF, seed=1))
    args = [t.to(DEV) for t in (q, k, v, *par, log_n_of(1, 170, 0))]
    want = apply_chord_attention_varlen(*args, ps, window=30, sinks=2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = apply_chord_attention_varlen(*args, ps, window=30, sinks=2)
    for _ in range(3):
        got.zero_()
        graph.replay()
        assert torch.equal(got, want)
        want = apply_chord_attention_varlen(*args, ps, window=30, sinks=2)


@pytest.mark.parametrize('dtype,D,L', [(BF, 64, 1), (BF, 64, 2), (F16, 64, 1), (F32, 128, 1), (BF, 32, 3)])
@torch.no_grad()
def test_cursor_step_appends_nothing_and_advances(dtype, D, L):
    from motif.ops.chord_attention import chord_decode_cursor, chord_window_workspace
    B, H, Hkv, cap, window, sinks = 2, 6, 2, 300, 50, 3
    _, k, v, par = inputs(B, H, Hkv, 1, cap, D, dtype, seed=L)
    table = torch.log(torch.arange(1, cap + 1, dtype=torch.float32))
    kd, vd = k.to(DEV), v.to(DEV)
    ws = chord_window_workspace(B, H, Hkv, L, cap, D, dtype, DEV, window, sinks)
    for cached in (0, 1, 49, 51, 200, cap - L):
        q, _, _, _ = inputs(B, H, Hkv, L, 1, D, dtype, seed=cached)
        cursor = torch.tensor([cached], dtype=torch.int32, device=DEV)
        got = chord_decode_cursor(q.to(DEV), kd, vd, cursor, *(t.to(DEV) for t in par), table.to(DEV), window=window,
                                  sinks=sinks, workspace=ws)
        assert int(cursor) == cached + L
        n = cached + L
        check_attention(got, q, k[:, :, :n], v[:, :, :n], par, table[cached:n][None].expand(B, L), cached, window, sinks,
                        what=f'cached {cached}')


@torch.no_grad()
def test_long_context_far_rows():
    '''Rows past 2^31 bytes from the start of the keys.'''
    S, L, window = 2 ** 18, 3, 4000
    g = torch.Generator(device=DEV).manual_seed(3)
    big = torch.randn(S, 72 * 64, generator=g, device=DEV, dtype=BF)  # 2.4 GB; row stride 4608
    k, v = big[None, None, :, :64], big[None, None, :, 64:128]
    q, _, _, par = inputs(1, 2, 1, L, 1, 64, BF, seed=1)
    log_n = log_n_of(1, L, S - L)
    got = _run(q, k, v, par, log_n, window=window, sinks=5)
    keep = list(range(5)) + list(range(S - L - window + 1, S))
    idx = torch.tensor(keep, device=DEV)
    # the same keys at their own positions: the reference over the kept rows alone
    kk, vv = k[:, :, idx].cpu().double(), v[:, :, idx].cpu().double()
    pos = torch.tensor(keep, dtype=torch.float64)
    al, be, mu, ss = (t.double().view(2, 1, 1) for t in par)
    d = pos[None] - (S - L + torch.arange(L)[:, None]).double()
    z = (q.double() @ kk.transpose(-1, -2) / 8 - al * ((d - mu).abs() + 1e-5) ** be) * (ss * log_n.double()[:, None, :, None])
    z = z.masked_fill(~((d <= 0) & ((d > -window) | (pos < 5)[None])), float('-inf'))
    p = torch.softmax(z, -1)
    lim = 2.0 ** -8 * (p @ vv.abs()) + 2.0 ** -8 * (p @ vv).abs() + 2.0 ** -11 * (p @ vv.abs())
    assert ((got.cpu().double() - p @ vv).abs() <= lim).all()


@torch.no_grad()
def test_window_that_covers_everything_equals_no_window_within_rounding():
    from motif.ops import apply_chord_attention
    q, k, v, par = inputs(1, 4, 2, 200, 200, 64, BF, seed=2)
    args = [t.to(DEV) for t in (q, k, v, *par, log_n_of(1, 200, 0))]
    out, _, allowed = attention64(q, k, v, par, log_n_of(1, 200, 0), 0)
    mean, _, _ = attention64(q, k, v.abs(), par, log_n_of(1, 200, 0), 0)
    a, b = apply_chord_attention(*args), apply_chord_attention(*args, window=200)
    h = 2.0 ** -8
    lim = 2 * (allowed + h * mean + h * out.abs()) + 2.0 ** -20
    assert ((a - b).double().abs().cpu() <= lim).all()


@torch.no_grad()
def test_captured_and_on_another_stream():
    from motif.ops import apply_chord_attention
    for shape in [(2, 4, 2, 1, 300, 299, 64, 64, 4), (1, 4, 2, 257, 257, 0, 64, 100, 3)]:
        B, H, Hkv, L, S, q_start, D, window, sinks = shape
        q, k, v, par = inputs(B, H, Hkv, L, S, D, BF, seed=1)
        args = [t.to(DEV) for t in (q, k, v, *par, log_n_of(B, L, q_start))]
        want = apply_chord_attention(*args, window=window, sinks=sinks)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = apply_chord_attention(*args, window=window, sinks=sinks)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = apply_chord_attention(*args, window=window, sinks=sinks)
        for seed in (7, 8, 9):
            q2, k2, v2, _ = inputs(B, H, Hkv, L, S, D, BF, seed=seed)
            for dst, src in zip(args[:3], (q2, k2, v2)):
                dst.copy_(src)
            graph.replay()
            assert torch.equal(got, apply_chord_attention(*args, window=window, sinks=sinks))


@pytest.mark.parametrize('dtype', [BF, F16, F32], ids=['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('L', [1, 3, 90])
@pytest.mark.parametrize('scale', [0.125, -0.125, 0.0])
@torch.no_grad()
def test_parameters_at_their_edges(dtype, L, scale):
    '''Heads with ssmax zero and negative, alpha zero and negative, beta zero and negative, mu on a key, and
    scales of either sign and zero.'''
    H, Hkv, S, window, sinks = 8, 2, 140, 45, 3
    q, k, v, par = inputs(2, H, Hkv, L, S, 64, dtype, seed=L)
    al, be, mu, ss = (t.clone() for t in par)
    ss[0], ss[1], ss[7] = 0.0, -ss[1], -ss[7]
    al[2], al[3] = 0.0, -al[3]
    be[4], be[5] = 0.0, -0.3
    mu[6], mu[7] = 0.0, -7.0
    par = (al, be, mu, ss)
    log_n = log_n_of(2, L, S - L)
    got = _run(q, k, v, par, log_n, window=window, sinks=sinks, softmax_scale=scale)
    check_attention(got, q, k, v, par, log_n, S - L, window, sinks, scale=scale)


@pytest.mark.parametrize('B', [1, 40])
@torch.no_grad()
def test_split_decode_of_rows_that_see_nothing(B):
    '''A window that ends past the keys, long enough to be split over workgroups: zeros.'''
    q, k, v, par = inputs(B, 4, 2, 2, 2000, 64, BF, seed=2)
    log_n = log_n_of(B, 2, 5000)
    assert not _run(q, k, v, par, log_n, q_start=5000, window=2000).any()
    got = _run(q, k, v, par, log_n, q_start=5000, window=2000, sinks=2)
    check_attention(got, q, k, v, par, log_n, 5000, 2000, 2)


@pytest.mark.parametrize('dtype', [BF, F16, F32], ids=['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('L', [2, 100])
@torch.no_grad()
def test_log_n_of_either_sign(dtype, L):
    S, window, sinks = 180, 45, 3
    q, k, v, par = inputs(2, 8, 2, L, S, 64, dtype, seed=L)
    log_n = log_n_of(2, L, S - L)
    log_n[0, ::2] *= -0.5
    log_n[1, L // 2:] = 0.0
    for scale in (0.125, -0.2, 0.0):
        got = _run(q, k, v, par, log_n, window=window, sinks=sinks, softmax_scale=scale)
        check_attention(got, q, k, v, par, log_n, S - L, window, sinks, scale=scale)


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
@torch.no_grad()
def test_long_context_far_rows_of_a_prefill(dtype):
    '''The same for many queries: rows past 2^31 bytes from the start of the keys, and more than 2^24 back.'''
    S, L, window, sinks = 2 ** 25, 70, 300, 5
    g = gen(4)
    k = torch.zeros(1, 1, S, 64, dtype=dtype, device=DEV)  # 4.3 GB (bf16), and as much for the values
    v = torch.zeros(1, 1, S, 64, dtype=dtype, device=DEV)
    rows = list(range(sinks)) + list(range(S - L - window, S))
    idx = torch.tensor(rows, device=DEV)
    for t in (k, v):
        t[:, :, idx] = torch.randn(1, 1, len(rows), 64, generator=g).to(dtype).to(DEV)
    q, _, _, par = inputs(1, 2, 1, L, 1, 64, dtype, seed=1)
    log_n = log_n_of(1, L, S - L)
    got = _run(q, k, v, par, log_n, window=window, sinks=sinks).cpu().double()
    want, mean = over_rows64(q, rows, k[:, :, idx], v[:, :, idx], par, log_n, S - L, window, sinks)
    # logits to 2^7, a weight to 2^-15 of itself by fp32's steps; bf16: P's and the output's rounding besides
    lim = 2.0 ** -14 * mean + ((2.0 ** -8 * mean + 2.0 ** -8 * want.abs()) if dtype == BF else 0)
    assert ((got - want).abs() <= lim).all()
