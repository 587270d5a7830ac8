'''Gradients of Chord attention under a window against the formula in float64 and against
differences, for the kernels (bf16, head dim 64) and the torch form (other types).'''
import pytest
import torch

from support import gen
from window_ref import inputs, log_n_of, seen

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF = torch.bfloat16


def formula64(q, k, v, par, log_n, do, q_start, window, sinks, eps=1e-5):
    '''(gradients [dq, dk, dv, dalpha, dbeta, dmu, dssmax], bounds of the kernels' distance).

    bf16 kernels round, with h = 2^-8 each: P and s c dZ where they enter a product, O where
    Delta = dO . O is formed (an error of h |dO| . |O| per row), and the result.  For the
    parameter gradients, which carry none of these, the bound takes 2^-15 of the sum of the
    terms' sizes (logits up to 2^6 in fp32: 2^-18, twice, for the weight and the row's sum;
    the bias's derivatives to 2^-18).'''
    q, k, v, do, log_n = (t.detach().cpu().double() for t in (q, k, v, do, log_n))
    al, be, mu, ss = (t.detach().cpu().double().view(-1, 1, 1) for t in par)
    B, H, L, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    G = H // Hkv
    kf, vf = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    d = (torch.arange(S)[None] - (q_start + torch.arange(L)[:, None])).double()
    x = (d - mu).abs() + eps
    xb = x ** be
    lam = log_n[:, None, :, None]
    c, s, h = ss * lam, D ** -0.5, 2.0 ** -8
    r = s * (q @ kf.transpose(-1, -2)) - al * xb
    keep = seen(L, S, q_start, window, sinks)
    P = torch.softmax((c * r).masked_fill(~keep, -1e300), -1) * keep
    O = P @ vf
    dP = do @ vf.transpose(-1, -2)
    dZ = P * (dP - (do * O).sum(-1, keepdim=True))
    cdz = c * dZ
    fold = lambda t: t.view(B, Hkv, G, S, D).sum(2)
    dq, dk, dv = s * cdz @ kf, fold(s * cdz.transpose(-1, -2) @ q), fold(P.transpose(-1, -2) @ do)
    terms = [-cdz * xb, -cdz * al * xb * x.log(), cdz * al * be * x ** (be - 1) * torch.sign(d - mu), lam * dZ * r]
    grads = [dq, dk, dv, *[t.sum((0, 2, 3)) for t in terms]]
    # an element of s c dZ is off by its own rounding and by Delta's: h |s c| P |dO| . |O|, and fp32's
    ez = s * (h * cdz.abs() + h * c.abs() * P * (do.abs() * O.abs()).sum(-1, keepdim=True)
              + 2.0 ** -13 * c.abs() * P * (dP.abs() + 1))
    lims = [ez @ kf.abs(), fold(ez.transpose(-1, -2) @ q.abs()), fold((h + 2.0 ** -13) * P.transpose(-1, -2) @ do.abs())]
    lims = [l + h * g.abs() + 1e-6 for l, g in zip(lims, grads)]
    lims += [2.0 ** -15 * (t.abs() + (P * w.abs() * dP.abs() * c.abs()).abs()).sum((0, 2, 3)) + 1e-6
             for t, w in zip(terms, (xb, al * xb * x.log(), al * be * x ** (be - 1), r / ss.abs().clamp_min(1e-9)))]
    return grads, lims


def _grads(q, k, v, par, log_n, do, q_start, window, sinks, dev=DEV):
    from motif.ops import apply_chord_attention
    xs = [t.to(dev).detach().requires_grad_() for t in (q, k, v, *par)]
    o = apply_chord_attention(*xs, log_n.to(dev), q_start=q_start, window=window, sinks=sinks)
    return o.detach(), torch.autograd.grad(o, xs, do.to(dev))


# B, H, Hkv, L, S, q_start, window, sinks
SHAPES = [
    (1, 1, 1, 1, 1, 0, 1, 0),
    (1, 2, 2, 5, 5, 0, 1, 0),            # a window of one key: constant rows, zero dq and dk
    (2, 4, 2, 33, 33, 0, 16, 0),
    (1, 4, 4, 130, 130, 0, 40, 3),
    (2, 4, 1, 300, 300, 0, 64, 1),
    (1, 12, 3, 257, 400, 143, 100, 130),  # first tokens over two key blocks
    (1, 4, 4, 700, 700, 0, 33, 5),       # chunks behind the window of the first block
    (1, 2, 1, 1500, 1500, 0, 40, 200),
    (1, 3, 3, 200, 200, 0, 1000, 0),
    (1, 2, 2, 90, 90, 0, 8, 500),
    (1, 2, 1, 200, 64, 0, 20, 0),        # rows that see nothing
    (1, 2, 2, 40, 16, 100, 16, 0),       # no row sees anything
    (1, 4, 2, 40, 16, 100, 16, 2),
    (1, 4, 2, 1, 300, 299, 100, 4),
    (2, 2, 2, 3, 500, 300, 100, 4),      # keys behind the last query
    (1, 4, 2, 480, 480, 0, 420, 2),      # a long window of few blocks
    (2, 2, 1, 100, 620, 520, 500, 0),
]


@pytest.mark.parametrize('shape', SHAPES, ids=[str(s) for s in SHAPES])
def test_against_the_formula(shape):
    B, H, Hkv, L, S, q_start, window, sinks = shape
    q, k, v, par = inputs(B, H, Hkv, L, S, 64, BF, seed=sum(shape))
    log_n = log_n_of(B, L, q_start)
    do = torch.randn(B, H, L, 64, generator=gen(1)).to(BF)
    want, lims = formula64(q, k, v, par, log_n, do, q_start, window, sinks)
    _, got = _grads(q, k, v, par, log_n, do, q_start, window, sinks)
    for name, g, w, lim in zip(('dq', 'dk', 'dv', 'dalpha', 'dbeta', 'dmu', 'dssmax'), got, want, lims):
        dist = (g.cpu().double() - w).abs()
        assert (dist <= lim).all(), f'{name}: worst {float((dist / lim).max()):.2f} of the limit'


def test_parameter_gradients_carry_no_bf16_rounding():
    q, k, v, par = inputs(2, 4, 2, 512, 512, 64, BF, seed=3)
    log_n = log_n_of(2, 512, 0)
    do = torch.randn(2, 4, 512, 64, generator=gen(1)).to(BF)
    want, _ = formula64(q, k, v, par, log_n, do, 0, 128, 4)
    _, got = _grads(q, k, v, par, log_n, do, 0, 128, 4)
    for g, w in zip(got[3:], want[3:]):
        assert float((g.cpu().double() - w).norm() / w.norm()) < 2e-5


@pytest.mark.parametrize('dtype,D', [(BF, 64), (torch.float32, 64), (torch.float16, 32)])
def test_against_differences(dtype, D):
    '''Directional derivatives of the float64 formula's output by central differences
    against the gradients' inner products.'''
    from motif.ops.autograd_path import chord_attention_torch
    B, H, Hkv, L, S, window, sinks = 1, 4, 2, 60, 90, 25, 2
    q, k, v, par = inputs(B, H, Hkv, L, S, D, dtype, seed=11)
    log_n = log_n_of(B, L, S - L)
    do = torch.randn(B, H, L, D, generator=gen(2)).to(dtype)
    _, got = _grads(q, k, v, par, log_n, do, S - L, window, sinks)
    xs = [t.double() for t in (q, k, v, *par)]
    f = lambda ys: (chord_attention_torch(*ys, log_n.double(), S - L, window=window, sinks=sinks) * do.double()).sum()
    g = gen(5)
    for i, x in enumerate(xs):
        way = torch.randn(x.shape, generator=g, dtype=torch.float64)
        h = 1e-5
        up, down = ([y + s * h * way if j == i else y for j, y in enumerate(xs)] for s in (1, -1))
        slope = float((f(up) - f(down)) / (2 * h))
        terms = (got[i].cpu().double() * way)
        # every element off by a few roundings of its type, in random directions
        step = torch.finfo(dtype).eps if i < 3 else 2.0 ** -14
        lim = 6 * step * float(terms.norm()) + 4 * step * float(got[i].double().norm()) + 1e-4
        assert abs(float(terms.sum()) - slope) <= lim, (i, float(terms.sum()), slope, lim)


def test_broadcast_and_strided_inputs():
    from motif.ops import apply_chord_attention
    B, H, Hkv, L, window, sinks = 3, 4, 2, 100, 30, 2
    q, k, v, par = inputs(1, H, Hkv, L, L, 64, BF, seed=4)
    log_n = log_n_of(B, L, 0)
    do = torch.randn(B, L, H, 64, generator=gen(1)).to(BF)
    xs = [t.to(DEV).detach().requires_grad_() for t in (q, k, v)]
    ps = [t.to(DEV) for t in par]
    # one set of keys for the whole batch: its gradient is the sum over the batch
    o = apply_chord_attention(xs[0].expand(B, H, L, 64), xs[1].expand(B, Hkv, L, 64), xs[2].expand(B, Hkv, L, 64), *ps,
                              log_n.to(DEV), window=window, sinks=sinks)
    got = torch.autograd.grad(o, xs, do.to(DEV).transpose(1, 2))
    want, lims = formula64(q.expand(B, -1, -1, -1), k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), par, log_n,
                           do.transpose(1, 2), 0, window, sinks)
    for g, w, lim in zip(got, want, lims):
        # (the sum over the batch in bf16: two more roundings)
        assert ((g.cpu().double() - w.sum(0, keepdim=True)).abs()
                <= lim.sum(0, keepdim=True) + 2.0 ** -7 * w.abs().sum(0, keepdim=True)).all()
    # gradients broadcast over rows, as of a mean, and of a transposed layout
    one = torch.randn(1, 1, 1, 64, generator=gen(3)).to(BF).to(DEV)
    a = _grads(q, k, v, par, log_n[:1], one.expand(1, H, L, 64), 0, window, sinks)[1]
    b = _grads(q, k, v, par, log_n[:1], one.expand(1, H, L, 64).contiguous(), 0, window, sinks)[1]
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_rows_that_no_query_sees_get_zero_whatever_they_hold():
    B, H, Hkv, L, S, window, sinks = 1, 4, 2, 70, 333, 50, 3
    q, k, v, par = inputs(B, H, Hkv, L, S, 64, BF, seed=6)
    log_n = log_n_of(B, L, S - L)
    do = torch.randn(B, H, L, 64, generator=gen(1)).to(BF)
    _, want = _grads(q, k, v, par, log_n, do, S - L, window, sinks)
    dead = slice(sinks, S - L - window + 1)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, dead] = float('nan')
    v2[:, :, dead] = float('inf')
    _, got = _grads(q, k2, v2, par, log_n, do, S - L, window, sinks)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert not got[1][:, :, dead].any() and not got[2][:, :, dead].any()


def test_repeats_bit_for_bit_and_only_what_is_asked_for():
    from motif.ops import apply_chord_attention
    q, k, v, par = inputs(2, 4, 4, 300, 300, 64, BF, seed=8)
    log_n = log_n_of(2, 300, 0)
    do = torch.randn(2, 4, 300, 64, generator=gen(1)).to(BF)
    a, b = (_grads(q, k, v, par, log_n, do, 0, 64, 5)[1] for _ in range(2))
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    qd = q.to(DEV).requires_grad_()
    o = apply_chord_attention(qd, k.to(DEV), v.to(DEV), *(t.to(DEV) for t in par), log_n.to(DEV), window=64, sinks=5)
    assert torch.equal(torch.autograd.grad(o, qd, do.to(DEV))[0], a[0])


def test_no_queries_or_no_keys():
    for L, S in ((0, 5), (4, 0)):
        q, k, v, par = inputs(1, 2, 1, L, S, 64, BF)
        _, got = _grads(q, k, v, par, log_n_of(1, L, 0), torch.zeros(1, 2, L, 64, dtype=BF), 0, 3, 0)
        for g in got:
            assert not g.any()


def test_packed_gradients_equal_sequences_apart():
    from motif.ops import apply_chord_attention, apply_chord_attention_varlen
    lens = [70, 1, 33]
    T = sum(lens)
    q, k, v, par = inputs(1, 4, 2, T, T, 64, BF, seed=9)
    log_n = torch.cat([log_n_of(1, n, 0) for n in lens], 1).to(DEV)
    cu = torch.tensor([0, 70, 71, 104], dtype=torch.int32, device=DEV)
    do = torch.randn(1, 4, T, 64, generator=gen(1)).to(BF).to(DEV)
    xs = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    ps = [t.to(DEV) for t in par]
    got = torch.autograd.grad(apply_chord_attention_varlen(*xs, *ps, log_n, cu, window=20, sinks=1), xs, do)
    for a, b in ((0, 70), (70, 71), (71, 104)):
        ys = [t.detach()[:, :, a:b].clone().requires_grad_() for t in xs]
        one = torch.autograd.grad(apply_chord_attention(*ys, *ps, log_n[:, a:b], window=20, sinks=1), ys, do[:, :, a:b])
        for g, w in zip(got, one):
            assert torch.equal(g[:, :, a:b], w)


def test_training_step_in_a_graph():
    '''Forward and backward captured together, replayed on new data.'''
    from motif.ops import apply_chord_attention
    q, k, v, par = inputs(1, 4, 2, 150, 150, 64, BF, seed=10)
    log_n = log_n_of(1, 150, 0).to(DEV)
    ps = [t.to(DEV) for t in par]
    xs = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    do = torch.randn(1, 4, 150, 64, generator=gen(1)).to(BF).to(DEV)

    def step():
        o = apply_chord_attention(*xs, *ps, log_n, window=40, sinks=2)
        return torch.autograd.grad(o, xs, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2, 3):
        new = inputs(1, 4, 2, 150, 150, 64, BF, seed=seed)[:3]
        with torch.no_grad():
            for x, y in zip(xs, new):
                x.copy_(y)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)



def test_parameters_at_their_edges():
    '''Heads with ssmax zero and negative, alpha zero and negative, beta zero and negative, mu on a key.'''
    H, Hkv, L, window, sinks = 8, 4, 150, 45, 3
    q, k, v, par = inputs(1, H, Hkv, L, L, 64, BF, seed=6)
    al, be, mu, ss = (t.clone() for t in par)
    ss[0], ss[1] = 0.0, -ss[1]
    al[2], al[3] = 0.0, -al[3]
    be[4], be[5] = 0.0, -0.3
    mu[6], mu[7] = 0.0, -7.0
    par = (al, be, mu, ss)
    log_n = log_n_of(1, L, 0)
    do = torch.randn(1, H, L, 64, generator=gen(1)).to(BF)
    _, got = _grads(q, k, v, par, log_n, do, 0, window, sinks)
    want, lims = formula64(q, k, v, par, log_n, do, 0, window, sinks)
    for n, a, b, lim in zip(('dq', 'dk', 'dv', 'dalpha', 'dbeta', 'dmu', 'dssmax'), got, want, lims):
        assert ((a.cpu().double() - b).abs() <= lim).all(), n


def test_every_token_a_first_token():
    q, k, v, par = inputs(1, 4, 2, 200, 200, 64, BF, seed=3)
    log_n, do = log_n_of(1, 200, 0), torch.randn(1, 4, 200, 64, generator=gen(2)).to(BF)
    o, a = _grads(q, k, v, par, log_n, do, 0, 10, 200)
    o2, b = _grads(q, k, v, par, log_n, do, 0, 1000, 0)
    assert torch.equal(o, o2) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_second_derivatives_are_refused():
    q, k, v, par = inputs(1, 2, 1, 20, 20, 64, BF, seed=3)
    from motif.ops import apply_chord_attention
    q = q.to(DEV).requires_grad_()
    o = apply_chord_attention(q, *(t.to(DEV) for t in (k, v, *par, log_n_of(1, 20, 0))), window=5)
    with pytest.raises(RuntimeError, match='second derivatives'):
        torch.autograd.grad(o.float().sum(), q, create_graph=True)


def test_log_n_of_either_sign():
    q, k, v, par = inputs(1, 4, 2, 140, 140, 64, BF, seed=8)
    log_n = log_n_of(1, 140, 0)
    log_n[0, ::3] *= -0.5
    log_n[0, 100:] = 0.0
    do = torch.randn(1, 4, 140, 64, generator=gen(2)).to(BF)
    _, got = _grads(q, k, v, par, log_n, do, 0, 40, 2)
    want, lims = formula64(q, k, v, par, log_n, do, 0, 40, 2)
    for n, a, b, lim in zip(('dq', 'dk', 'dv', 'dalpha', 'dbeta', 'dmu', 'dssmax'), got, want, lims):
        assert ((a.cpu().double() - b).abs() <= lim).all(), n
