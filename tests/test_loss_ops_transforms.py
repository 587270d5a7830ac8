'''linear_cross_entropy, the row norms and dropout_add under what cannot follow their kernels: tracing, function transforms
and forward-mode derivatives are refused, instead of a result without its tangent or a trace of an empty tensor.'''
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from motif.ops import dropout_add, layer_norm_rows, linear_cross_entropy, rms_norm_rows

W, T, V = torch.ones(8), torch.tensor([1, 0, 3, 2, -100, 5]), torch.linspace(-1, 1, 80).view(10, 8)
OPS = {
    'linear_cross_entropy': lambda x: linear_cross_entropy(x, V.to(x.device), T.to(x.device)),
    'rms_norm_rows': lambda x: rms_norm_rows(x, W.to(x.device)),
    'layer_norm_rows': lambda x: layer_norm_rows(x, W.to(x.device), W.to(x.device)),
    'dropout_add': lambda x: dropout_add(x, 0.5, 3, residual=x),
}
# the same with the value of interest in another place
PLACES = {
    'linear_cross_entropy': lambda w: linear_cross_entropy(torch.ones(6, 8, device=w.device), w.view(6, 8), T.to(w.device) % 6),
    'rms_norm_rows': lambda w: rms_norm_rows(torch.ones(6, 8, device=w.device), w[0]),
    'layer_norm_rows': lambda w: layer_norm_rows(torch.ones(6, 8, device=w.device), W.to(w.device), w[0]),
    'dropout_add': lambda w: dropout_add(torch.ones(6, 8, device=w.device), 0.5, 3, residual=w),
}
DEVICES = pytest.mark.parametrize('device', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
BOTH = pytest.mark.parametrize('ops', [OPS, PLACES], ids=['first', 'other'])
NAMES = pytest.mark.parametrize('name', list(OPS))


def _x(device):
    return torch.linspace(-1, 2, 48, device=device).view(6, 8)


@DEVICES
@BOTH
@NAMES
def test_forward_mode_is_refused(name, ops, device):
    x = _x(device)
    with fwAD.dual_level():
        dual = fwAD.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match=f'{name}.*forward-mode'):
            ops[name](dual)


@DEVICES
@NAMES
def test_tracing_is_refused(name, device):
    with pytest.raises(NotImplementedError, match=f'{name}.*traced'):
        torch.jit.trace(OPS[name], (_x(device),))


@DEVICES
@NAMES
def test_symbolic_tracing_is_refused(name, device):
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(NotImplementedError, match=f'{name}.*traced'):
        make_fx(OPS[name])(_x(device))


@DEVICES
@BOTH
@NAMES
def test_function_transforms_are_refused(name, ops, device):
    x = _x(device)
    for run in (lambda: torch.func.grad(lambda t: ops[name](t).sum())(x),
                lambda: torch.func.vmap(ops[name])(torch.stack([x, x])),
                lambda: torch.func.jvp(ops[name], (x,), (x,))):
        with pytest.raises(NotImplementedError, match=f'{name}.*(function transform|forward-mode)'):
            run()


@DEVICES
def test_a_seed_of_its_own_for_each_is_refused(device):
    x, seeds = _x(device), torch.arange(2, device=device)
    with pytest.raises(NotImplementedError, match='dropout_add.*function transform'):
        torch.func.vmap(lambda s: dropout_add(x, 0.5, s))(seeds)


@pytest.mark.gpu
@NAMES
def test_plain_tensors_inside_a_dual_level(name):
    x = _x('cuda')
    want = OPS[name](x)
    with fwAD.dual_level():
        assert torch.equal(OPS[name](x), want)


@pytest.mark.gpu
def test_norm_module_keeps_its_tangent():
    from motif.ops import RMSNorm
    norm = RMSNorm(8).to('cuda')
    x, t = _x('cuda'), torch.linspace(1, -1, 48, device='cuda').view(6, 8)
    with fwAD.dual_level():
        y, got = fwAD.unpack_dual(norm(fwAD.make_dual(x, t)))
    x64, t64 = x.double(), t.double()
    r = 1 / torch.sqrt(x64.square().mean(-1, keepdim=True) + norm.eps)
    want = r * (t64 - x64 * r * r * (x64 * t64).mean(-1, keepdim=True))
    # sums of 8 terms and some ten operations in fp32
    assert got is not None and (got.double() - want).abs().max() <= 30 * 2.0 ** -24 * want.abs().max()


@pytest.mark.gpu
@NAMES
def test_a_gradient_with_a_tangent(name):
    '''A forward-mode tangent on the gradient that comes in, its input without one: linear through the norms, refused by the others.'''
    x = _x('cuda').requires_grad_()
    y = OPS[name](x)
    dy, t = torch.full_like(y, 0.5), torch.full_like(y, -2.0) if y.dim() == 0 else torch.cos(torch.arange(y.numel(), device='cuda') * 1.0).view(y.shape)
    want, = torch.autograd.grad(y, x, t, retain_graph=True)
    with fwAD.dual_level():
        dual = fwAD.make_dual(dy, t)
        if 'norm' not in name:
            with pytest.raises(NotImplementedError, match=f'{name}.*forward-mode'):
                torch.autograd.grad(y, x, dual)
            return
        got = fwAD.unpack_dual(torch.autograd.grad(y, x, dual)[0]).tangent
    # fp32 on both ways: two sums of eight terms and some twenty operations
    assert got is not None and (got - want).abs().max() <= 60 * 2.0 ** -24 * want.abs().max()


@pytest.mark.gpu
def test_model_loss_is_not_traced():
    from motif.model.config import MotifChordConfig
    from motif.model.motif import MotifChordModel
    cfg = MotifChordConfig(vocab_size=32, model_dim=64, num_heads=2, num_kv_heads=1, head_k_dim=32, block=('gdn', 'chord'), block_n=1)
    model = MotifChordModel(cfg).to('cuda').eval().requires_grad_(False)
    ids = torch.arange(6, device='cuda').view(1, 6)
    with torch.no_grad(), pytest.raises(NotImplementedError, match='linear_cross_entropy.*traced'):
        torch.jit.trace(lambda t: model(t, labels=t, fused_loss=True).loss, (ids,), check_trace=False)


@pytest.mark.gpu
@NAMES
def test_a_compiled_caller(name):
    '''torch.compile leaves the graph for the call.'''
    x = _x('cuda')
    torch._dynamo.reset()
    got = torch.compile(lambda t: OPS[name](t * 2) + 1, backend='eager')(x)
    assert torch.equal(got, OPS[name](x * 2) + 1)
