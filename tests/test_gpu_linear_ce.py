'''linear_cross_entropy against its float64 form: losses and gradients over sizes, types, strides,
rows without labels and bad labels; streams, graphs, repeats.'''
import pytest
import torch

from loss_ref import ce64, check

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF, F32 = torch.bfloat16, torch.float32


def _op():
    from motif.ops import linear_cross_entropy
    return linear_cross_entropy


def _inputs(N, d, V, dtype, ignored=0.0, seed=0, boost=10.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (0.05 * torch.randn(V, d, generator=g, device=DEV)).to(dtype)
    labels = torch.randint(0, V, (N,), generator=g, device=DEV)
    t = w[labels].float()
    a = boost * torch.rand(N, 1, generator=g, device=DEV)
    x = (torch.randn(N, d, generator=g, device=DEV) + a * t / t.pow(2).sum(-1, keepdim=True).clamp_min(0.01)).to(dtype)
    labels = torch.where(torch.rand(N, generator=g, device=DEV) < ignored, -100, labels)
    return x, w, labels


def _run(x, w, labels, reduction='mean', dloss=None, **kw):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = _op()(x, w, labels, reduction=reduction, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), dloss))


def _check(x, w, labels, reduction='mean', dloss=None):
    if dloss is None:
        dloss = torch.ones((), device=DEV)
    got = _run(x, w, labels, reduction, dloss)
    want = ce64(x, w, labels, dloss, reduction)
    for m, what in enumerate(('loss', 'dx', 'dw')):
        check(got[m], want[2 * m], want[2 * m + 1], what)
    return got


SIZES = [(1, 8, 1), (1, 64, 257), (2, 1, 3), (3, 100, 300), (65, 72, 255), (127, 64, 129), (128, 128, 256), (129, 200, 1000),
         (256, 256, 4097), (257, 768, 5003), (300, 1000, 513), (1025, 96, 8191), (40, 768, 32000)]


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('N,d,V', SIZES)
def test_mean_and_gradients(N, d, V, dtype):
    _check(*_inputs(N, d, V, dtype, seed=N + d))


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('N,d,V', [(1, 64, 300), (130, 64, 300), (515, 136, 2049)])
def test_sum_and_rows(N, d, V, dtype):
    x, w, labels = _inputs(N, d, V, dtype, ignored=0.4, seed=5)
    g = torch.Generator(device=DEV).manual_seed(1)
    _check(x, w, labels, 'sum', torch.tensor(0.37, device=DEV))
    _check(x, w, labels, 'none', torch.randn(N, generator=g, device=DEV))
    _check(x, w, labels, 'none', torch.ones(1, device=DEV).expand(N))
    _check(x, w, labels, 'none', torch.randn(2 * N, generator=g, device=DEV)[::2])


@pytest.mark.parametrize('d,V', [(256, 40960), (768, 40001)])
def test_large_training_step(d, V):
    '''Several vocabulary pieces (P of a piece holds 256 MB and more) and full tiles.'''
    _check(*_inputs(8192 + 77, d, V, BF, ignored=0.1, seed=2))


def test_several_pieces_in_fp32():
    _check(*_inputs(8192 + 5, 64, 9001, F32, ignored=0.05, seed=4))


def test_many_rows_of_a_small_vocabulary():
    _check(*_inputs(70001, 64, 500, BF, ignored=0.2, seed=3))


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
def test_large_logits(dtype):
    '''Confident rows: one z far above the others, and all far below zero.'''
    x, w, labels = _inputs(200, 64, 700, dtype, seed=6)
    _check(x * 30, w, labels)
    w2 = w.clone()
    w2[:, 0] = -8
    x2 = x.clone()
    x2[:, 0] = 40
    _check(x2, w2, labels)


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
def test_ignored_rows_reach_nothing(dtype):
    x, w, labels = _inputs(300, 72, 900, dtype, ignored=0.5, seed=7)
    clean = _run(x, w, labels)
    x2 = x.clone()
    bad = labels == -100
    x2[bad] = float('nan')
    x2[bad.nonzero()[0]] = float('inf')
    for got, want in zip(_run(x2, w, labels), clean):
        assert torch.equal(got, want)
    assert not clean[1][bad].any()


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
def test_no_label_at_all(dtype):
    x, w, labels = _inputs(70, 64, 300, dtype, seed=8)
    labels = torch.full_like(labels, 7)
    for red in ('mean', 'sum', 'none'):
        dl = torch.ones(70, device=DEV) if red == 'none' else torch.ones((), device=DEV)
        loss, dx, dw = _run(x, w, labels, red, dl, ignore_index=7)
        assert not dx.any() and not dw.any()
        assert bool(loss.isnan()) if red == 'mean' else not loss.any()


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('bad', [-1, 300, 2 ** 40])
def test_label_outside_the_vocabulary(bad, dtype):
    x, w, labels = _inputs(140, 64, 300, dtype, seed=9)
    loss, dx, _ = _run(x, w, labels, 'none', torch.ones(140, device=DEV))
    labels[77] = bad
    loss2, dx2, dw2 = _run(x, w, labels, 'none', torch.ones(140, device=DEV))
    keep = torch.arange(140, device=DEV) != 77
    assert torch.equal(loss[keep], loss2[keep]) and torch.equal(dx[keep], dx2[keep])
    assert bool(loss2[77].isnan()) and bool(dx2[77].isnan().all()) and bool(dw2.isnan().all())
    assert bool(_op()(x, w, labels).isnan())


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
def test_vocabulary_rows_of_minus_infinity(dtype):
    '''A word that no row may choose, in the middle and for whole tiles.'''
    x, w, labels = _inputs(130, 64, 1000, dtype, seed=10)
    x[:, 0] = 1
    w2 = w.clone()
    w2[0:400, 0] = float('-inf')
    w2[999, 0] = float('-inf')
    labels = labels % 500 + 450
    got = _op()(x, w2, labels, reduction='none')
    keep = torch.ones(1000, dtype=torch.bool, device=DEV)
    keep[0:400] = keep[999] = False
    want, tol = ce64(x, w2[keep], labels - 400, reduction='none')
    check(got, want, tol, 'loss')


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
def test_strides_and_alignment(dtype):
    x, w, labels = _inputs(150, 64, 333, dtype, ignored=0.2, seed=11)
    want = _run(x, w, labels)

    def same(x, w, labels, exact=True):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = _op()(x, w, labels)
        for got, ref in zip((loss.detach(), *torch.autograd.grad(loss, (x, w))), want):
            if exact:
                assert torch.equal(got, ref)
            else:  # (another kernel: the bounds of both)
                check(got, ref.double(), 2e-2 * ref.double().abs().max() if dtype == BF else 2e-5 * ref.double().abs().max(), 'x')
    wide = torch.empty(150, 200, dtype=dtype, device=DEV)
    wide[:, 8:72] = x
    same(wide[:, 8:72], w, labels)          # a row stride, aligned
    wide[:, 3:67] = x
    same(wide[:, 3:67], w, labels)          # off 16 bytes
    same(x.t().contiguous().t(), w, labels)  # features apart
    lab2 = torch.stack([labels, labels], 1)
    same(x, w, lab2[:, 0])
    same(x, w, labels.to(torch.int32))
    ww = torch.empty(333, 72, dtype=dtype, device=DEV)
    ww[:, :64] = w
    same(x, ww[:, :64], labels)
    ww[:, 1:65] = w
    same(x, ww[:, 1:65], labels, exact=dtype == F32)
    ww = torch.empty(333, 67, dtype=dtype, device=DEV)
    ww[:, :64] = w
    same(x, ww[:, :64], labels, exact=dtype == F32)
    x3, l3 = x.view(3, 50, 64), labels.view(3, 50)
    loss = _op()(x3, w, l3, reduction='none')
    assert loss.shape == (3, 50)
    assert torch.equal(loss.flatten(), _op()(x, w, labels, reduction='none'))


def test_row_shared_by_all_tokens():
    '''A broadcast input: its gradient is the sum over the rows.'''
    x, w, labels = _inputs(60, 64, 300, F32, seed=12)
    row = x[:1].detach().requires_grad_()
    loss = _op()(row.expand(60, 64), w, labels)
    got, = torch.autograd.grad(loss, (row,))
    want = ce64(x[:1].expand(60, 64), w, labels, torch.ones((), device=DEV))
    check(got, want[2].sum(0, keepdim=True), want[3].sum(0, keepdim=True) * 2, 'dx')


def test_offsets_past_32_bits():
    '''Rows of x and of the vocabulary that lie 2^31 elements apart.'''
    far = 2 ** 30 + 8
    x, w, labels = _inputs(3, 64, 3, BF, seed=13)
    want = _run(x, w, labels)
    buf = torch.empty(3 * far, dtype=BF, device=DEV)
    xf = buf.as_strided((3, 64), (far, 1))
    xf.copy_(x)
    wf = buf.as_strided((3, 64), (far, 1), 64)
    wf.copy_(w)
    got = _run(xf, wf, labels)
    assert torch.equal(got[0], want[0]) or abs(got[0] - want[0]) < 1e-5
    ref = ce64(x, w, labels, torch.ones((), device=DEV))
    check(got[1], ref[2], ref[3], 'dx')
    check(got[2], ref[4], ref[5], 'dw')


def test_gradient_of_one_input_alone():
    x, w, labels = _inputs(200, 128, 1000, BF, ignored=0.1, seed=14)
    _, dx, dw = _run(x, w, labels)
    xg = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(_op()(xg, w, labels), xg)[0], dx)
    wg = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(_op()(x, wg, labels), wg)[0], dw)


def test_gradients_against_differences():
    '''Central differences of the float64 loss along random directions.'''
    x, w, labels = _inputs(20, 40, 90, F32, ignored=0.2, seed=15)
    _, dx, dw = _run(x, w, labels)
    g = torch.Generator(device=DEV).manual_seed(3)
    for _ in range(4):
        ux, uw = (torch.randn(t.shape, generator=g, device=DEV, dtype=torch.float64) for t in (x, w))
        e = 1e-5
        hi = ce64(x.double() + e * ux, w.double() + e * uw, labels)[0]
        lo = ce64(x.double() - e * ux, w.double() - e * uw, labels)[0]
        want = (hi - lo) / (2 * e)
        got = (dx.double() * ux).sum() + (dw.double() * uw).sum()
        # truncation e^2 |f'''| (f''' of order |u|^3 ~ 1e4 here: 1e-6), cancellation 1e-16 / 1e-5, gradients to 1e-5
        assert abs(got - want) <= 1e-4 * max(1.0, abs(float(want)))


def test_repeats_bit_for_bit_and_on_another_stream():
    x, w, labels = _inputs(1500, 256, 9000, BF, ignored=0.1, seed=16)
    want = _run(x, w, labels)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(_run(x, w, labels), want))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _run(x, w, labels)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_step_replays():
    op = _op()
    xs, w, ls = _inputs(600, 128, 3001, BF, ignored=0.2, seed=17)
    x, labels = xs.detach().clone().requires_grad_(), ls.clone()
    w = w.detach().requires_grad_()

    def step():
        loss = op(x, w, labels)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (18, 19, 20, 21):  # (other rows without labels each time)
        x2, _, l2 = _inputs(600, 128, 3001, BF, ignored=0.1 * (seed - 17), seed=seed)
        with torch.no_grad():
            x.copy_(x2)
        labels.copy_(l2)
        graph.replay()
        torch.cuda.synchronize()
        want = _run(x2, w, l2)
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_autocast_casts_as_linear():
    x, w, labels = _inputs(100, 64, 500, F32, seed=22)
    with torch.autocast('cuda', dtype=BF):
        got = _op()(x, w, labels)
    assert torch.equal(got, _op()(x.to(BF), w.to(BF), labels))


def test_no_rows():
    w = torch.randn(10, 8, device=DEV, requires_grad=True)
    x = torch.empty(0, 8, device=DEV, requires_grad=True)
    t = torch.empty(0, dtype=torch.int64, device=DEV)
    assert bool(_op()(x, w, t).isnan())
    assert _op()(x, w, t, reduction='none').shape == (0,)
    s = _op()(x, w, t, reduction='sum')
    s.backward()
    assert float(s.detach()) == 0 and not w.grad.any() and x.grad.shape == (0, 8)


def test_second_derivatives_are_refused():
    x, w, labels = _inputs(10, 16, 20, F32, seed=23)
    x.requires_grad_()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(_op()(x, w, labels), x, create_graph=True)
