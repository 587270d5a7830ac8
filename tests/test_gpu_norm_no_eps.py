'''RMSNorm without an eps in training: torch's own op, which then takes the type's.'''
import pytest
import torch
import torch.nn.functional as F

from support import gen

pytestmark = pytest.mark.gpu

DEV = 'cuda'


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_training_without_an_eps(dtype):
    from motif.ops import RMSNorm
    norm = RMSNorm(64, eps=None).to(DEV, dtype)
    x = torch.randn(10, 64, generator=gen(1)).to(DEV, dtype).requires_grad_()
    dy = torch.randn(10, 64, generator=gen(2)).to(DEV, dtype)

    def train(f):
        y = f(x)
        return (y.detach(), *torch.autograd.grad(y, (x, norm.weight), dy))
    got = train(norm)
    want = train(lambda t: F.rms_norm(t, (64,), norm.weight, None))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        assert torch.equal(norm(x), want[0])


def test_the_operator_needs_one():
    from motif.ops import layer_norm_rows, rms_norm_rows
    x = torch.ones(3, 8, device=DEV)
    for fn in (rms_norm_rows, layer_norm_rows):
        with pytest.raises(TypeError):
            fn(x, eps=None)
