'''Dropout of a residual branch whose mask is drawn again instead of stored
(csrc/dropout.hip; the reference has no dropout).
'''
import torch

from . import _lib
from .autograd_path import refuse_transforms


def dropout_add(x, p, seed, residual=None):
    '''residual + x * keep / (1 - p) (without a residual: x * keep / (1 - p)), x and residual of
    one shape and dtype (fp32, bf16 or fp16), computed in fp32 and rounded once; a dropped
    element adds nothing, whatever x holds there.

    Element e of x (its row-major index) is kept when word e mod 4 of Philox4x32-10 at counter
    e div 4 under the 64-bit key `seed` is at least round(p 2^32), 0 <= p < 1.  `seed` is an int, or
    an int64 tensor of one element on x's device that is read when the kernel runs (so that a
    captured graph draws anew when it changes); it must stay as it is until the backward.
    Differentiable once in x and residual, in reverse mode; tracing, function transforms and
    forward-mode tangents are refused.'''
    refuse_transforms('dropout_add', x, residual, seed if isinstance(seed, torch.Tensor) else None)
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
        seed = (seed + 2 ** 63) % 2 ** 64 - 2 ** 63  # (its 64 bits as an int64)
    else:
        raise TypeError(f'dropout_add: seed must be an int or an int64 tensor, got {type(seed).__name__}')
    if not x.is_cuda:
        raise ValueError(f'dropout_add: x is on {x.device}, the kernels need a ROCm device')
    if isinstance(seed, int):
        return _lib.nodes().dropout_add(x, residual, p, seed, None)
    return _lib.nodes().dropout_add(x, residual, p, 0, seed)
