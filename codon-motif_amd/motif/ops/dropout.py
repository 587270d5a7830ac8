'''Dropout of a residual branch whose mask is drawn again instead of stored
(csrc/dropout.hip; the reference has no dropout).
'''
import torch

from . import _lib


def _launch(x, residual, p, seed):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    n = x.numel()
    if n == 0:
        return y
    threshold = min(int(round(p * 2 ** 32)), 2 ** 32 - 1)
    value, dev_seed = (0, seed.data_ptr()) if isinstance(seed, torch.Tensor) else (seed, None)
    with _lib.on_device(x.device):
        rc = _lib.lib().motif_dropout_add(x.data_ptr(), _lib.ptr(residual), y.data_ptr(), n, threshold, 1 / (1 - p),
                                          value, dev_seed, _lib.chord_dtype_code(x.dtype), _lib.stream_ptr(x.device))
    if rc:
        _lib.check(rc, 'motif_dropout_add')
    return y


class DropoutAddFunction(torch.autograd.Function):
    '''motif_dropout_add; its backward draws the forward's words again.'''

    @staticmethod
    def forward(ctx, x, residual, p, seed):
        on_device = isinstance(seed, torch.Tensor)
        ctx.save_for_backward(*((seed,) if on_device else ()))
        ctx.p, ctx.seed = p, None if on_device else seed
        return _launch(x.contiguous(), None if residual is None else residual.contiguous(), p, seed)

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():  # (create_graph: what the kernel gives carries no graph)
            raise RuntimeError('dropout_add has no second derivatives')
        seed = ctx.saved_tensors[0] if ctx.seed is None else ctx.seed
        dx = _launch(dy.contiguous(), None, ctx.p, seed) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None


def dropout_add(x, p, seed, residual=None):
    '''residual + x * keep / (1 - p) (without a residual: x * keep / (1 - p)), x and residual of
    one shape and dtype (fp32, bf16 or fp16), computed in fp32 and rounded once; a dropped
    element adds nothing, whatever x holds there.

    Element e of x (its row-major index) is kept when word e mod 4 of Philox4x32-10 at counter
    e div 4 under the 64-bit key `seed` is at least round(p 2^32), 0 <= p < 1.  `seed` is an int, or
    an int64 tensor of one element on x's device that is read when the kernel runs (so that a
    captured graph draws anew when it changes); it must stay as it is until the backward.
    Differentiable once in x and residual.'''
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise ValueError(f'dropout_add: p must be in [0, 1), got {p}')
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise NotImplementedError(f'dropout_add: unsupported dtype {x.dtype}')
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f'dropout_add: residual must be {tuple(x.shape)} of {x.dtype} on {x.device}, got '
                         f'{tuple(residual.shape)} of {residual.dtype} on {residual.device}')
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != x.device:
            raise ValueError(f'dropout_add: a seed tensor holds one int64 on {x.device}')
    elif isinstance(seed, int) and not isinstance(seed, bool):
        if not -2 ** 63 <= seed < 2 ** 64:
            raise ValueError('dropout_add: the seed has 64 bits')
        seed &= 2 ** 64 - 1
    else:
        raise TypeError(f'dropout_add: seed must be an int or an int64 tensor, got {type(seed).__name__}')
    if not x.is_cuda:
        raise ValueError(f'dropout_add: x is on {x.device}, the kernels need a ROCm device')
    return DropoutAddFunction.apply(x, residual, p, seed)
