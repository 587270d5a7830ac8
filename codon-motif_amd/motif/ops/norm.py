'''RMSNorm and LayerNorm of rows with their gradients (csrc/row_norm.hip).

The forward of the reference's row norms (motif/ops/rms_norm.py:17-61) in one pass over
fp32 arithmetic, rounded once, and their backward (:63-112) with the weight's gradient
summed in a fixed order.  `RMSNorm` calls `rms_norm_rows` where gradients are wanted.
'''
import torch

from . import _lib
from .autograd_path import refuse_transforms

MAX_FEATURES = 16384
_DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _check(x, params, what):
    refuse_transforms(what, x, *(t for _, t in params))
    if x.dtype not in _DTYPES:
        raise NotImplementedError(f'{what}: unsupported dtype {x.dtype}')
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f'{what}: x needs features, got {tuple(x.shape)}')
    D = x.shape[-1]
    if D > MAX_FEATURES:
        raise NotImplementedError(f'{what}: at most {MAX_FEATURES} features, got {D}')
    if x.numel() // D >= 2 ** 31:
        raise ValueError(f'{what}: too many rows')
    for name, t in params:
        if t is None:
            continue
        if t.shape != (D,) or t.dtype != x.dtype or t.device != x.device:
            raise ValueError(f'{what}: {name} must be [{D}] of {x.dtype} on {x.device}, got {tuple(t.shape)} of '
                             f'{t.dtype} on {t.device}')
    if not x.is_cuda:
        raise ValueError(f'{what}: x is on {x.device}, the kernels need a ROCm device')


def rms_norm_rows(x, weight=None, eps=1e-6):
    '''x / sqrt(mean(x^2) + eps) * weight over the last dimension of x [..., D] (fp32, bf16 or
    fp16, D at most 16384), in fp32, rounded once.  weight [D] of x's dtype, or None.
    Differentiable in x and weight, in
    reverse mode; tracing, function transforms and forward-mode tangents are refused.'''
    _check(x, (('weight', weight),), 'rms_norm_rows')
    return _lib.nodes().row_norm(x, weight, None, eps, False)


def layer_norm_rows(x, weight=None, bias=None, eps=1e-5):
    '''(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x [..., D], as
    rms_norm_rows; bias [D] of x's dtype, or None.  Differentiable in x, weight and bias in
    the same way.'''
    _check(x, (('weight', weight), ('bias', bias)), 'layer_norm_rows')
    return _lib.nodes().row_norm(x, weight, bias, eps, True)
