'''The loss from the hidden states, the row norms and dropout from several streams, threads and
captured graphs at once, and inside a checkpointed function: each equals the same work alone.'''
import threading

import pytest
import torch

from support import gen

pytestmark = pytest.mark.gpu

DEV = 'cuda'
SIZES = [(3000, 256, 9000, 0.1), (1000, 128, 5000, 0.3)]  # tokens, features, words, share ignored


def _inputs(i):
    N, d, V, ignored = SIZES[i]
    g = gen(i + 1)
    x = torch.randn(N, d, generator=g).to(DEV, torch.bfloat16).requires_grad_()
    w = (torch.randn(V, d, generator=g) * 2 * d ** -0.5).to(DEV, torch.bfloat16).requires_grad_()
    labels = torch.randint(0, V, (N,), generator=g)
    labels[torch.rand(N, generator=g) < ignored] = -100
    return x, w, labels.to(DEV), torch.full((d,), 0.9, device=DEV, dtype=torch.bfloat16, requires_grad=True)


def _step(x, w, labels, scale):
    '''Norm, dropout and loss with their gradients.'''
    from motif.ops import dropout_add, linear_cross_entropy, rms_norm_rows
    h = dropout_add(rms_norm_rows(x, scale), 0.2, 77, residual=x)
    loss = linear_cross_entropy(h, w, labels)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w, scale)))


def _same(got, want):
    return all(torch.equal(u, v) for u, v in zip(got, want))


def test_two_streams():
    a, b = _inputs(0), _inputs(1)
    alone = _step(*a), _step(*b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            p = _step(*a)
        with torch.cuda.stream(s2):
            q = _step(*b)
        torch.cuda.synchronize()
        assert _same(p, alone[0]) and _same(q, alone[1])


def test_threads():
    a = _inputs(0)
    alone = _step(*a)
    torch.cuda.synchronize()
    got = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(3):
                out = _step(*a)
            torch.cuda.current_stream().synchronize()
        got[i] = out

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 4 and all(_same(out, alone) for out in got.values())


def test_two_captured_graphs():
    '''Two graphs share nothing: replayed at once on two streams, with eager steps between.'''
    inputs = _inputs(0), _inputs(1)
    alone = [_step(*a) for a in inputs]
    graphs, outs = [], []
    for a in inputs:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(*a)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(*a)
        graphs.append(graph)
        outs.append(out)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(_same(out, want) for out, want in zip(outs, alone))
        assert _same(_step(*inputs[1]), alone[1])
        torch.cuda.synchronize()


def test_checkpointed():
    '''A seed drawn from torch's generator is drawn again when the function runs again.'''
    from torch.utils.checkpoint import checkpoint

    from motif.ops import dropout_add, rms_norm_rows
    t = torch.randn(100, 64, generator=gen(3)).to(DEV).requires_grad_()
    w = torch.full((64,), 1.1, device=DEV, requires_grad=True)

    def f(t):
        seed = torch.randint(2 ** 63 - 1, (1,), device=DEV)
        return dropout_add(rms_norm_rows(t, w), 0.3, seed, residual=t)

    def run(g):
        torch.manual_seed(0)
        y = g(t)
        return (y.detach(), *torch.autograd.grad(y.sum(), (t, w)))

    assert _same(run(lambda t: checkpoint(f, t, use_reentrant=False)), run(f))


@pytest.mark.parametrize('which', ['loss', 'norm', 'dropout'])
def test_captured_beside_a_held_loss(which):
    '''A backward captured while an eager graph of the same leaves lives is refused before the leaf's
    default stream is made to wait for the capture; without that graph it is captured.'''
    from motif.ops import dropout_add, linear_cross_entropy, rms_norm_rows
    x, w, labels, scale = _inputs(1)

    def forward():
        if which == 'loss':
            return linear_cross_entropy(x, w, labels)
        if which == 'norm':
            return rms_norm_rows(x, scale)
        return dropout_add(x, 0.3, 5)

    leaf = {'loss': w, 'norm': scale, 'dropout': x}[which]
    held = forward()
    seed = torch.ones_like(held)
    want = torch.autograd.grad(held, leaf, seed, retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='still held'):
        with torch.cuda.graph(graph):
            torch.autograd.grad(forward(), leaf, seed)
    torch.cuda.synchronize()
    assert _same(torch.autograd.grad(held, leaf, seed, retain_graph=True), want)  # (eager work goes on)
    held = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(forward(), leaf, seed)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert _same(out, want)
