'''dropout_add against its definition: which elements are kept, values and gradients.'''
import pytest
import torch

from loss_ref import U, check, half, kept

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DTYPES = pytest.mark.parametrize('dtype', [BF, F16, F32], ids=['bf16', 'fp16', 'fp32'])


def _op():
    from motif.ops import dropout_add
    return dropout_add


def _inputs(shape, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(shape, generator=g, device=DEV).to(dtype) for _ in range(3)]


def _check(shape, dtype, p, seed, key=None):
    x, res, dy = _inputs(shape, dtype, 3)
    keep = kept(x.numel(), key if key is not None else seed % 2 ** 64, p).to(DEV).view(shape)
    for r in (None, res):
        xg = x.detach().requires_grad_()
        rg = None if r is None else r.detach().requires_grad_()
        y = _op()(xg, p, seed, residual=rg)
        grads = torch.autograd.grad(y, (xg,) if r is None else (xg, rg), dy)
        f = keep.double() / (1 - p)
        base = 0 if r is None else r.double()
        want = base + x.double() * f
        tol = half(dtype) * want.abs() + 4 * U * (x.double().abs() * f + (0 if r is None else r.double().abs())) \
            + torch.finfo(dtype).tiny
        check(y, want, tol, 'y')
        assert torch.equal(grads[0] != 0, keep & (dy != 0))
        check(grads[0], dy.double() * f, (half(dtype) + 4 * U) * (dy.double() * f).abs() + torch.finfo(dtype).tiny, 'dx')
        if r is not None:
            assert torch.equal(grads[1], dy)


@DTYPES
@pytest.mark.parametrize('shape', [(1,), (3,), (4,), (7,), (8,), (9,), (255,), (33, 65), (64, 768), (2, 5, 7, 11), (300, 1001)])
def test_values_and_gradients(shape, dtype):
    _check(shape, dtype, 0.3, 1234567890123456789)


@pytest.mark.parametrize('p', [0.0, 1e-6, 0.1, 0.5, 0.9, 0.999, 1 - 1e-12])
def test_probabilities(p):
    if p > 0.99999:  # (all but a word of ones dropped)
        x = torch.ones(5000, device=DEV)
        assert not _op()(x, p, 5).any()
        assert torch.equal(_op()(x, p, 5, residual=x), x)
        return
    _check((20011,), BF, p, 99)


@pytest.mark.parametrize('seed', [0, -1, 2 ** 63, 2 ** 64 - 1, 2 ** 32, -2 ** 63])
def test_seeds(seed):
    _check((1003,), F32, 0.4, seed)


def test_seed_on_the_device():
    _check((1003,), BF, 0.4, torch.tensor([-12345], device=DEV), key=-12345 % 2 ** 64)
    _check((1003,), BF, 0.4, torch.tensor(7, device=DEV), key=7)


def test_seed_changed_before_the_backward_is_an_error():
    x = torch.randn(100, device=DEV, requires_grad=True)
    seed = torch.tensor([3], device=DEV)
    y = _op()(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_share_kept():
    '''Of n words, n (1 - p) are kept up to six standard deviations.'''
    n, p = 1 << 22, 0.1
    got = int((_op()(torch.ones(n, device=DEV), p, 77) != 0).sum())
    assert abs(got - n * (1 - p)) <= 6 * (n * p * (1 - p)) ** 0.5


@DTYPES
def test_dropped_elements_add_nothing(dtype):
    x, res, dy = _inputs((4000,), dtype, 4)
    keep = kept(4000, 21, 0.5).to(DEV)
    want = _op()(x, 0.5, 21, residual=res)
    x2 = torch.where(keep, x, torch.full_like(x, float('nan')))
    assert torch.equal(_op()(x2, 0.5, 21, residual=res), want)
    xg = x.detach().requires_grad_()
    dx, = torch.autograd.grad(_op()(xg, 0.5, 21), xg, torch.where(keep, dy, torch.full_like(dy, float('inf'))))
    assert not dx[~keep].any()


@DTYPES
def test_strides_and_alignment(dtype):
    x, res, dy = _inputs((40, 72), dtype, 5)
    want = _op()(x, 0.25, 8, residual=res)
    assert torch.equal(_op()(x.t().contiguous().t(), 0.25, 8, residual=res), want)
    off = torch.empty(40 * 72 + 3, dtype=dtype, device=DEV)
    xo = off[3:].view(40, 72)
    xo.copy_(x)
    assert torch.equal(_op()(xo, 0.25, 8, residual=res), want)
    xg = x.detach().requires_grad_()
    a, = torch.autograd.grad(_op()(xg, 0.25, 8), xg, dy)
    b, = torch.autograd.grad(_op()(xg, 0.25, 8), xg, dy.t().contiguous().t())
    assert torch.equal(a, b)
    c, = torch.autograd.grad(_op()(xg, 0.25, 8).sum(), xg)  # (an expanded gradient)
    assert torch.equal(c != 0, kept(40 * 72, 8, 0.25).to(DEV).view(40, 72))


def test_elements_past_32_bits():
    '''More than 2^34 elements: the counter's second word counts.'''
    n = 2 ** 34 + 4 * 1000
    x = torch.ones(n, dtype=BF, device=DEV)
    y = _op()(x, 0.5, 31)
    del x
    for first in (0, 2 ** 31, 2 ** 32, 2 ** 34 - 2000, 2 ** 34):
        assert torch.equal(y[first:first + 4000].cpu() != 0, kept(4000, 31, 0.5, first)), first


def test_no_elements():
    x = torch.empty(0, 5, device=DEV, requires_grad=True)
    y = _op()(x, 0.5, 1)
    y.sum().backward()
    assert y.shape == (0, 5) and x.grad.shape == (0, 5)


def test_stream_and_captured_step_with_a_moving_seed():
    x, res, dy = _inputs((500, 96), BF, 6)
    want = _op()(x, 0.2, 50, residual=res)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _op()(x, 0.2, 50, residual=res)
    s.synchronize()
    assert torch.equal(got, want)
    seed = torch.tensor([50], device=DEV)
    xg = x.detach().clone().requires_grad_()

    def step():
        y = _op()(xg, 0.2, seed, residual=res)
        return y.detach(), torch.autograd.grad(y, xg, dy)[0]
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for value in (50, 51, -3, 2 ** 40):
        seed.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        keep = kept(x.numel(), value % 2 ** 64, 0.2).to(DEV).view(x.shape)
        assert torch.equal(out[0], _op()(x, 0.2, value, residual=res))
        assert torch.equal(out[1] != 0, keep & (dy != 0))


def test_second_derivatives_are_refused():
    x = torch.randn(10, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(_op()(x, 0.5, 1).sum(), x, create_graph=True)
