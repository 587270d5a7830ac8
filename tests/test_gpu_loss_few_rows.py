'''linear_cross_entropy in bf16 with up to 32 labelled rows: nothing of the logits' gradient is lost to bf16 before the
products, so the gradients are as close to float64 as their own rounding allows.'''
import pytest
import torch

from loss_ref import ce64, check, half

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF = torch.bfloat16


def _inputs(N, d, V, labelled, seed, boost=10.0):
    '''N rows of which `labelled`, spread over them, have a label; some are confident of it, some are not.'''
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (0.05 * torch.randn(V, d, generator=g, device=DEV)).to(BF)
    labels = torch.randint(0, V, (N,), generator=g, device=DEV)
    t = w[labels].float()
    a = boost * torch.rand(N, 1, generator=g, device=DEV)
    x = (torch.randn(N, d, generator=g, device=DEV) + a * t / t.pow(2).sum(-1, keepdim=True).clamp_min(0.01)).to(BF)
    keep = torch.randperm(N, generator=g, device=DEV)[:labelled]
    mask = torch.full_like(labels, -100)
    mask[keep] = labels[keep]
    return x, w, mask


def _run(x, w, labels, reduction='mean', dloss=None):
    from motif.ops import linear_cross_entropy
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = linear_cross_entropy(x, w, labels, reduction=reduction)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), dloss))


def _check(x, w, labels, reduction='mean', dloss=None):
    dloss = torch.ones((), device=DEV) if dloss is None else dloss
    got = _run(x, w, labels, reduction, dloss)
    # bounds of a computation in fp32 throughout, and on them one rounding of the result and two to bf16's remainder of P: 2^-16 of it
    loss, t_loss, dx, t_dx, dw, t_dw = ce64(x.float(), w.float(), labels, dloss, reduction)
    live = labels != -100
    z = x[live].double() @ w.double().t()
    P = z.softmax(-1)
    P[torch.arange(len(P), device=DEV), labels[live]] -= 1
    s = dloss.double().expand(len(labels))[live] if reduction == 'none' else dloss.double() / (max(len(P), 1) if reduction == 'mean' else 1)
    P = (P * (s[:, None] if reduction == 'none' else s)).abs()
    t_dx, t_dw = t_dx + half(BF) * dx.abs(), t_dw + half(BF) * dw.abs()
    t_dx[live] += 2.0 ** -16 * (P @ w.double().abs())
    t_dw += 2.0 ** -16 * (P.t() @ x[live].double().abs())
    check(got[0], loss, t_loss, 'loss')
    check(got[1], dx, t_dx, 'dx')
    check(got[2], dw, t_dw, 'dw')
    return got


@pytest.mark.parametrize('labelled', [1, 2, 3, 8, 15, 16, 17, 31, 32])
@pytest.mark.parametrize('d,V', [(64, 257), (100, 5003), (768, 4099)])
def test_few_rows(labelled, d, V):
    _check(*_inputs(labelled, d, V, labelled, seed=labelled))


@pytest.mark.parametrize('N,d,V,labelled', [(33, 64, 700, 32), (129, 64, 700, 32), (300, 72, 2049, 5), (2560, 512, 3001, 27), (3000, 768, 40000, 32), (9000, 64, 513, 20)])
def test_few_labels_among_many_rows(N, d, V, labelled):
    '''The same from the count on the device, under every tile that the sizes choose.'''
    _check(*_inputs(N, d, V, labelled, seed=N))


@pytest.mark.parametrize('reduction', ['none', 'sum'])
def test_reductions(reduction):
    x, w, labels = _inputs(200, 136, 999, 30, seed=3)
    g = torch.Generator(device=DEV).manual_seed(1)
    _check(x, w, labels, reduction, torch.randn(200, generator=g, device=DEV) if reduction == 'none' else torch.tensor(-0.37, device=DEV))


def test_several_pieces_of_the_vocabulary():
    '''70000 rows lay P out in pieces of 4096 words or little more.'''
    _check(*_inputs(70000, 64, 9001, 30, seed=4))


def test_unaligned_words():
    x, w, labels = _inputs(30, 72, 600, 30, seed=5)
    wide = torch.empty(600, 75, dtype=BF, device=DEV)
    wide[:, 1:73] = w
    _check(x, wide[:, 1:73], labels)


def test_a_gradient_that_is_no_number_stays_in_its_row():
    x, w, labels = _inputs(30, 64, 300, 30, seed=6)
    dl = torch.ones(30, device=DEV)
    clean = _run(x, w, labels, 'none', dl)
    for bad in (float('inf'), float('nan')):
        dl[11] = bad
        dx = _run(x, w, labels, 'none', dl)[1]
        keep = torch.arange(30, device=DEV) != 11
        assert torch.equal(dx[keep], clean[1][keep]) and not bool(dx[11].isfinite().any())


def test_replays_across_the_border():
    '''A captured step whose labels come and go follows the count from one way to the other.'''
    from motif.ops import linear_cross_entropy
    x, w, labels = _inputs(400, 128, 3001, 400, seed=7)
    x, w = x.requires_grad_(), w.requires_grad_()
    now = labels.clone()

    def step():
        loss = linear_cross_entropy(x, w, now)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in (400, 32, 33, 1, 300, 5, 0, 31):
        now.copy_(torch.where(torch.arange(400, device=DEV) % 400 < n, labels, -100))
        graph.replay()
        torch.cuda.synchronize()
        want = _run(x, w, now)
        assert all(bool(((a == b) | (a.isnan() & b.isnan())).all()) for a, b in zip(out, want)), n
