'''rms_norm_rows and layer_norm_rows against their float64 forms, forward and backward.'''
import pytest
import torch

from loss_ref import check, norm64

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DTYPES = pytest.mark.parametrize('dtype', [BF, F16, F32], ids=['bf16', 'fp16', 'fp32'])
LAYER = pytest.mark.parametrize('layer', [0, 1], ids=['rms', 'layer'])


def _op(layer):
    from motif.ops import layer_norm_rows, rms_norm_rows
    return (lambda x, w=None, b=None, eps=1e-5: layer_norm_rows(x, w, b, eps)) if layer else (
        lambda x, w=None, b=None, eps=1e-5: rms_norm_rows(x, w, eps))


def _inputs(N, D, dtype, seed=0, shift=0.3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)
    return ((1.5 * rnd(N, D) + shift).to(dtype), (1 + 0.2 * rnd(D)).to(dtype), (0.2 * rnd(D)).to(dtype), rnd(N, D).to(dtype))


def _run(layer, x, w, b, dy, eps=1e-5):
    leaves = [t for t in (x, w, b if layer else None) if t is not None]
    leaves = [t.detach().requires_grad_() for t in leaves]
    it = iter(leaves)
    x, w, b = next(it), None if w is None else next(it), next(it) if layer and b is not None else None
    y = _op(layer)(x, w, b, eps)
    return [y.detach(), *torch.autograd.grad(y, leaves, dy)]


def _check(layer, x, w, b, dy, eps=1e-5):
    got = _run(layer, x, w, b, dy, eps)
    want = norm64(x, w, b if layer else None, dy, eps, layer)
    want = want[:2] + ([want[2]] if w is not None else []) + ([want[3]] if layer and b is not None else [])
    for m, (g, (v, t)) in enumerate(zip(got, want)):
        check(g, v, t, ('y', 'dx', 'dw', 'db')[m])
    return got


WIDTHS = [1, 2, 7, 8, 16, 63, 64, 65, 100, 128, 256, 257, 768, 771, 1024, 1025, 1536, 2048, 2050, 4096, 4100, 8192, 16383, 16384]


@LAYER
@DTYPES
@pytest.mark.parametrize('D', WIDTHS)
def test_widths(D, dtype, layer):
    _check(layer, *_inputs(5 if D > 2000 else 37, D, dtype, seed=D))


@LAYER
@pytest.mark.parametrize('N,D', [(1, 768), (2, 64), (1023, 768), (9001, 64), (20000, 128), (1500, 771), (5000, 16)])
def test_many_rows(N, D, layer):
    '''More rows than one step of the backward's grid, and a last step that is not full.'''
    _check(layer, *_inputs(N, D, BF, seed=N))
    if N * D < 10 ** 6:
        _check(layer, *_inputs(N, D, F32, seed=N))


@LAYER
def test_without_weight_or_bias(layer):
    x, w, b, dy = _inputs(33, 96, F32, seed=1)
    _check(layer, x, None, None, dy)
    if layer:
        _check(layer, x, w, None, dy)
        _check(layer, x, None, b, dy)


@LAYER
def test_extreme_rows(layer):
    '''Rows of zeros, of one value, and of sizes near the square roots of fp32's ends.'''
    x, w, b, dy = _inputs(6, 64, F32, seed=2)
    x[0] = 0
    x[1] = 4.0
    x[2] *= 1e15
    x[3] *= 1e-12
    _check(layer, x, w, b, dy, 1e-6)


@LAYER
def test_a_row_of_no_number_stays_alone(layer):
    x, w, b, dy = _inputs(40, 72, BF, seed=3)
    clean = _op(layer)(x, w, b)
    x[17, 3] = float('nan')
    x[23, 0] = float('inf')
    got = _op(layer)(x, w, b)
    keep = [i for i in range(40) if i not in (17, 23)]
    assert torch.equal(got[keep], clean[keep]) and bool(got[17].isnan().all())


@LAYER
@DTYPES
def test_strides_and_alignment(dtype, layer):
    x, w, b, dy = _inputs(48, 64, dtype, seed=4)
    want = _run(layer, x, w, b, dy)
    n64 = norm64(x, w, b if layer else None, dy, 1e-5, layer)

    def same(x, w, b, dy, exact=True):
        for m, (g, r) in enumerate(zip(_run(layer, x, w, b, dy), want)):
            if exact:
                assert torch.equal(g.reshape(r.shape), r)
            else:
                check(g.reshape(r.shape), *n64[m], 'one element an access')
    wide = torch.zeros(48, 200, dtype=dtype, device=DEV)
    wide[:, 16:80] = x
    same(wide[:, 16:80], w, b, dy)
    wide[:, 1:65] = x
    same(wide[:, 1:65], w, b, dy, False)
    wide[:, 17:81] = dy
    same(x, w, b, wide[:, 17:81], False)
    same(x.t().contiguous().t(), w, b, dy)
    same(x, w, b, dy.t().contiguous().t())
    ww = torch.empty(65, dtype=dtype, device=DEV)
    ww[1:] = w
    same(x, ww[1:], b, dy, False)
    w2 = torch.stack([w, w], 1)
    same(x, w2[:, 0], b, dy)
    # [B, T, H, D] seen as [B, H, T, D]: the heads of a projection
    x4, dy4 = x.view(2, 4, 6, 64), dy.view(2, 4, 6, 64)
    got = _run(layer, x4.transpose(1, 2), w, b, dy4.transpose(1, 2))
    assert torch.equal(got[0].transpose(1, 2).reshape(48, 64), want[0])
    assert torch.equal(got[1].transpose(1, 2).reshape(48, 64), want[1])
    one = dy[:1].expand(48, 64)
    check(_run(layer, x, w, b, one)[1], *norm64(x, w, b if layer else None, one, 1e-5, layer)[1], 'dy of one row')


@LAYER
def test_broadcast_input(layer):
    x, w, b, _ = _inputs(1, 64, F32, seed=5)
    row = x.detach().requires_grad_()
    dy = _inputs(30, 64, F32, seed=6)[3]
    y = _op(layer)(row.expand(30, 64), w, b)
    got, = torch.autograd.grad(y, (row,), dy)
    v, t = norm64(x.expand(30, 64), w, b if layer else None, dy, 1e-5, layer)[1]
    check(got, v.sum(0, keepdim=True), 2 * t.sum(0, keepdim=True), 'dx')


@LAYER
def test_gradients_alone_and_no_rows(layer):
    x, w, b, dy = _inputs(50, 128, BF, seed=7)
    full = _run(layer, x, w, b, dy)
    wg = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(_op(layer)(x, wg, b), wg, dy)[0], full[2])
    xg = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(_op(layer)(xg, w, b), xg, dy)[0], full[1])
    if layer:
        bg = b.detach().requires_grad_()
        assert torch.equal(torch.autograd.grad(_op(layer)(x, w, bg), bg, dy)[0], full[3])
    out = _run(layer, x[:0], w, b, dy[:0])
    assert out[0].shape == (0, 128) and not out[2].any()
    assert _op(layer)(x[:0], w, b).shape == (0, 128)
    assert _op(layer)(x[3], w, b).shape == (128,)
    assert torch.equal(_op(layer)(x, w, b), full[0])  # (no gradients: the same values)


@LAYER
def test_gradients_against_differences(layer):
    x, w, b, dy = _inputs(6, 20, F32, seed=8)
    got = _run(layer, x, w, b, dy)
    g = torch.Generator(device=DEV).manual_seed(1)
    ins = (x, w, b) if layer else (x, w)
    dirs = [torch.randn(t.shape, generator=g, device=DEV, dtype=torch.float64) for t in ins]
    e = 1e-5

    def f(s):
        moved = [t.double() + s * u for t, u in zip(ins, dirs)] + [None] * (3 - len(ins))
        return (norm64(*moved, dy, 1e-5, layer)[0][0] * dy.double()).sum()
    want = (f(e) - f(-e)) / (2 * e)
    have = sum((t.double() * u).sum() for t, u in zip(got[1:], dirs))
    # truncation e^2 |f'''| ~ 1e-7, fp32 gradients to 1e-5 of their sizes
    assert abs(have - want) <= 1e-3


@LAYER
def test_offsets_past_32_bits(layer):
    N, D = 2 ** 25 + 5, 64
    x = torch.empty(N, D, dtype=BF, device=DEV)
    xs, w, b, dys = _inputs(7, D, BF, seed=9)
    x.zero_()
    x[-7:] = xs
    y = _op(layer)(x, w, b)
    assert torch.equal(y[-7:], _op(layer)(xs, w, b))
    del y
    dy = torch.zeros_like(x)
    dy[-7:] = dys
    xg = x.requires_grad_()
    got, = torch.autograd.grad(_op(layer)(xg, w, b), xg, dy)
    assert torch.equal(got[-7:], _run(layer, xs, w, b, dys)[1])


@LAYER
def test_repeats_streams_and_graphs(layer):
    x, w, b, dy = _inputs(3000, 768, BF, seed=10)
    want = _run(layer, x, w, b, dy)
    assert all(torch.equal(p, q) for p, q in zip(_run(layer, x, w, b, dy), want))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _run(layer, x, w, b, dy)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    xs = x.clone()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run(layer, xs, w, b, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(layer, xs, w, b, dy)
    for seed in (11, 12, 13):
        x2 = _inputs(3000, 768, BF, seed=seed)[0]
        xs.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, _run(layer, x2, w, b, dy)))


@LAYER
def test_second_derivatives(layer):
    '''The derivative of the gradients, against float64 torch ops.'''
    def norm(x, w, b):
        c = x - x.mean(-1, keepdim=True) if layer else x
        return c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5) * w + (b if layer else 0)

    def second(fn, x, w, b, dy):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        gx, gw = torch.autograd.grad(fn(x, w, b), (x, w), dy, create_graph=True)
        return torch.autograd.grad(gx.square().sum() + gw.square().sum(), (x, w))
    x, w, b, dy = _inputs(12, 40, F32, seed=14)
    got = second(_op(layer), x, w, b, dy)
    want = second(norm, x.double(), w.double(), b.double(), dy.double())
    for g, v in zip(got, want):
        # sums of 40 and of 12 terms in fp32, three deep: 1e-5 of the largest leaves a factor of ten
        assert (g.double() - v).abs().max() <= 1e-5 * v.abs().max()
