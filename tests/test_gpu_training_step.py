'''The row norms, dropout and the loss from the hidden states on the model's own paths: RMSNorm in
training, a decoder's dropped branches, the fused loss, and all of them in one captured step.'''
import copy

import pytest
import torch
import torch.nn.functional as F

from loss_ref import ce64, check, kept, norm64
from support import gen

pytestmark = pytest.mark.gpu

DEV = 'cuda'
BF, F32 = torch.bfloat16, torch.float32


def _model(dtype, seed=5, **kw):
    from motif.model.config import MotifChordConfig
    from motif.model.motif import MotifChordModel
    from motif.model.presets import init_random
    cfg = MotifChordConfig(vocab_size=160, model_dim=256, num_heads=4, num_kv_heads=2, head_k_dim=64,
                           block=('gdn', 'chord'), block_n=2, **kw)
    return init_random(MotifChordModel(cfg), std=0.05, seed=seed).to(DEV, dtype)


def _batch(B=2, T=96, seed=0, ignored=0.3):
    g = gen(seed)
    ids = torch.randint(0, 160, (B, T), generator=g)
    labels = torch.randint(0, 160, (B, T), generator=g)
    labels[torch.rand(B, T, generator=g) < ignored] = -100
    return ids.to(DEV), labels.to(DEV)


def _grads(model):
    return {n: p.grad for n, p in model.named_parameters() if p.grad is not None}


@pytest.mark.parametrize('dtype', [BF, torch.float16, F32], ids=['bf16', 'fp16', 'fp32'])
def test_rms_norm_module(dtype):
    from motif.ops import RMSNorm
    norm = RMSNorm(768).to(DEV, dtype)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.1 * torch.randn(768, generator=gen(1)))
    x = torch.randn(3, 50, 768, generator=gen(2)).to(DEV, dtype).requires_grad_()
    dy = torch.randn(3, 50, 768, generator=gen(3)).to(DEV, dtype)
    y = norm(x)
    got = torch.autograd.grad(y, (x, norm.weight), dy)
    want = norm64(x.view(-1, 768), norm.weight, None, dy.view(-1, 768), norm.eps, 0)
    check(y.view(-1, 768), *want[0], 'y')
    check(got[0].view(-1, 768), *want[1], 'dx')
    check(got[1], *want[2], 'dw')
    with torch.no_grad():  # (inference keeps torch's op: the same formula, a rounding apart at most)
        assert torch.equal(norm(x), F.rms_norm(x, (768,), norm.weight, norm.eps))


def test_rms_norm_module_elsewhere():
    '''Function transforms, autocast and mixed types keep torch's own op.'''
    from motif.ops import RMSNorm
    norm = RMSNorm(64).to(DEV)
    x = torch.randn(5, 64, device=DEV)
    g = torch.func.grad(lambda t: norm(t).square().sum())(x)
    xr = x.clone().requires_grad_()
    want, = torch.autograd.grad(norm(xr).square().sum(), xr)
    assert torch.allclose(g, want, rtol=1e-4, atol=1e-4)
    with torch.autocast('cuda', dtype=BF):
        assert norm(xr).shape == x.shape
    traced = torch.jit.trace(norm, (x,))
    assert torch.allclose(traced(2 * x + 1), norm(2 * x + 1), rtol=1e-5, atol=1e-5)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        assert norm(dual).shape == x.shape
    assert norm(x.to(BF).requires_grad_()).shape == x.shape
    assert norm(x[:, ::2].repeat(1, 2)).shape == x.shape


def test_fused_loss_equals_the_logits_loss():
    model = _model(F32, tied_weight=False)
    ids, labels = _batch()
    out = model(ids, labels=labels)
    out.loss.backward()
    want = {n: g.clone() for n, g in _grads(model).items()}
    ref = float(out.loss.detach())
    del out
    model.zero_grad()
    out = model(ids, labels=labels, fused_loss=True)
    assert out.logits is None and out.loss.dtype == F32
    dh, dw = torch.autograd.grad(out.loss, (out.hidden_states, model.lm_head.weight), retain_graph=True)
    h64 = ce64(out.hidden_states.detach().view(-1, 256), model.lm_head.weight, labels.view(-1), torch.ones((), device=DEV))
    check(out.loss, h64[0], h64[1], 'loss')
    check(dh.reshape(-1, 256), h64[2], h64[3], 'gradient of the hidden states')
    check(dw, h64[4], h64[5], "gradient of the vocabulary's rows")
    # F.cross_entropy over fp32 logits: the same bounds again
    assert abs(float(out.loss.detach()) - ref) <= 2 * float(h64[1])
    out.loss.backward()
    got = _grads(model)
    assert set(got) == set(want)
    # The two routes differ in the hidden states' gradient by some 1e-6 of it, and everything before them is linear in that.
    # Over all parameters together: single ones (an attention's alpha: 1e-8, the rest of sums that cancel) may be all rounding.
    far = sum((got[n] - want[n]).double().square().sum() for n in want) ** 0.5
    size = sum(want[n].double().square().sum() for n in want) ** 0.5
    assert far <= 1e-4 * size
    with torch.no_grad():
        assert torch.equal(model(ids, labels=labels, fused_loss=True).loss, out.loss.detach())


def test_bf16_training_step_descends():
    '''A step along the gradients that the kernels give lowers the loss by what they predict (first order).'''
    model = _model(BF)
    master = _model(F32)
    master.load_state_dict({k: v.float() for k, v in model.state_dict().items()})
    ids, labels = _batch(T=64)
    model(ids, labels=labels, fused_loss=True).loss.backward()
    grads = {n: g.float() for n, g in _grads(model).items()}
    master(ids, labels=labels, fused_loss=True).loss.backward()
    exact = _grads(master)
    dot = sum((grads[n] * exact[n]).sum() for n in exact)
    size = sum(exact[n].square().sum() for n in exact)
    other = sum(grads[n].square().sum() for n in exact)
    # (bf16 weights and activations: a whole gradient within some percent; at a right angle it would be 0)
    assert float(dot / (size * other).sqrt()) > 0.98


def test_dropout_only_in_training_and_by_the_seed():
    model = _model(F32, dropout=0.3)
    plain = _model(F32)
    ids, labels = _batch()
    with torch.no_grad():
        assert torch.equal(model.eval()(ids).logits, plain.eval()(ids).logits)
        model.train()
        torch.manual_seed(3)
        a = model(ids).logits
        torch.manual_seed(3)
        b = model(ids).logits
        c = model(ids).logits
        assert torch.equal(a, b) and not torch.equal(a, c)
    torch.manual_seed(3)
    d = model(ids, labels=labels)
    assert (d.logits.detach() - a).abs().max() <= 1e-3  # (the same elements dropped with gradients on)
    torch.manual_seed(3)
    assert abs(float(model(ids, labels=labels, fused_loss=True).loss.detach()) - float(d.loss.detach())) <= 1e-5


def test_dropped_branches():
    from motif.block.decoder import _dropped_branches
    a, m = (torch.randn(4, 300, 256, generator=gen(i)).to(DEV) for i in (1, 2))
    torch.manual_seed(8)
    f = _dropped_branches(0.25, a, m)
    torch.manual_seed(8)
    seeds = torch.randint(2 ** 63 - 1, (2,), device=DEV)
    ka, km = (kept(a.numel(), int(s), 0.25).to(DEV).view(a.shape) for s in seeds)
    want = a.double() * ka / 0.75 + m.double() * km / 0.75
    assert (f.double() - want).abs().max() <= 1e-6 * 10
    assert torch.equal((f == 0), ~(ka | km))
    assert _dropped_branches(0.5, a.cpu(), m.cpu()).shape == a.shape
    assert _dropped_branches(0.5, a, m.to(BF)).dtype == F32


def test_dropout_with_packed_sequences():
    model = _model(F32, dropout=0.2).train()
    ids, labels = _batch(1, 90)
    cu = torch.tensor([0, 30, 31, 90], dtype=torch.int32, device=DEV)
    torch.manual_seed(1)
    a = model(ids, cu_seqlens=cu, labels=labels, fused_loss=True).loss
    a.backward()
    torch.manual_seed(1)
    b = model(ids, cu_seqlens=cu, labels=labels).loss
    assert abs(float(a.detach()) - float(b.detach())) <= 1e-5
    assert all(torch.isfinite(g).all() for g in _grads(model).values())


@pytest.mark.parametrize('dtype', [BF, F32], ids=['bf16', 'fp32'])
def test_captured_training_step(dtype):
    '''Forward, fused loss and backward with dropout in one graph: every replay draws from the device's generator as
    an eager step from the same state does.'''
    model = _model(dtype, dropout=0.1).train()
    eager = copy.deepcopy(model)
    ids, labels = _batch(T=64)

    def step(m):
        for p in m.parameters():
            p.grad = None
        loss = m(ids, labels=labels, fused_loss=True).loss
        loss.backward()
        return loss.detach()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(model)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(model)
    seen = set()
    for seed in (1, 2, 3):
        torch.cuda.manual_seed(seed)
        want = step(eager)
        torch.cuda.manual_seed(seed)
        graph.replay()
        torch.cuda.synchronize()
        seen.add(float(loss))
        assert torch.equal(loss, want), (seed, float(loss), float(want))
        a, b = _grads(model), _grads(eager)
        for n in b:
            assert torch.isfinite(a[n]).all(), n
            assert (a[n] - b[n]).abs().max() <= 1e-6 * b[n].abs().max() + 1e-30, n
    assert len(seen) == 3
