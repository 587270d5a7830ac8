'''A step of the model along the gradients of its fused loss changes the loss as they predict; and the nodes with their saved
tensors moved to the host and back.'''
import pytest
import torch

from support import gen

pytestmark = pytest.mark.gpu

DEV = 'cuda'


def _model(seed=7):
    from motif.model.config import MotifChordConfig
    from motif.model.motif import MotifChordModel
    from motif.model.presets import init_random
    cfg = MotifChordConfig(vocab_size=160, model_dim=256, num_heads=4, num_kv_heads=2, head_k_dim=64, block=('gdn', 'chord'), block_n=1)
    return init_random(MotifChordModel(cfg), std=0.05, seed=seed).to(DEV)


def test_a_step_changes_the_loss_as_the_gradients_predict():
    model = _model()
    ids = torch.randint(0, 160, (2, 48), generator=gen(1)).to(DEV)
    labels = torch.randint(0, 160, (2, 48), generator=gen(2)).to(DEV)
    model(ids, labels=labels, fused_loss=True).loss.backward()
    params = [p for p in model.parameters() if p.grad is not None]
    size = sum(p.grad.double().square().sum() for p in params).sqrt()
    e = 1e-2
    losses = []
    with torch.no_grad():
        for sign in (1, -2):  # (to +e, then to -e)
            for p in params:
                p += (sign * e / size) * p.grad
            losses.append(float(model(ids, labels=labels, fused_loss=True).loss))
    got = (losses[0] - losses[1]) / (2 * e)
    # The loss of some 5 is good to 5 x 50 x 2^-24 = 1.5e-5: 1.5e-3 of the difference quotient; the third derivative along a
    # direction of length one stays within some hundreds of the first for weights of 0.05: e^2 / 6 of it, 1%.
    assert abs(got - float(size)) <= 1.5e-3 + 0.02 * float(size)


def test_saved_tensors_on_the_host():
    from motif.ops import dropout_add, layer_norm_rows, linear_cross_entropy
    x = torch.randn(300, 64, generator=gen(3)).to(DEV, torch.bfloat16).requires_grad_()
    wide = torch.randn(500, 72, generator=gen(4)).to(DEV, torch.bfloat16).requires_grad_()
    scale = torch.full((64,), 1.25, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    labels = torch.randint(0, 500, (300,), generator=gen(5)).to(DEV)
    seed = torch.tensor([3], device=DEV)

    def step():
        h = dropout_add(layer_norm_rows(x, scale, scale), 0.1, seed, residual=x)
        loss = linear_cross_entropy(h, wide[:, :64], labels)
        return (loss.detach(), *torch.autograd.grad(loss, (x, wide, scale)))
    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
