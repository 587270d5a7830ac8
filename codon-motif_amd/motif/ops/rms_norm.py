'''RMSNorm / GatedRMSNorm modules (adjacent to the hot path; PyTorch-ROCm).

Same parameters and formulas as the reference (motif/ops/rms_norm.py:419-553):
RMSNorm y = x / sqrt(mean(x^2) + eps) * weight; GatedRMSNorm takes
[values || gate] and returns rms_norm(values) * SiLU(gate).  Where gradients are wanted,
RMSNorm runs the HIP kernels of `rms_norm_rows` (the same formula, rounded once).
'''
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib
from .autograd_path import wants_grad
from .norm import MAX_FEATURES, rms_norm_rows

_KERNEL_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_PLAIN = (torch.Tensor, nn.Parameter)


def _trains_on_kernels(x, weight):
    '''A call whose gradients the kernels give: plain tensors in reverse mode.  Autocast, function
    transforms, forward-mode derivatives, tracing and compiling keep torch's own op, and so does an
    installation whose autograd nodes do not load.'''
    return (wants_grad(x, weight) and torch._C._get_tracing_state() is None and x.dtype in _KERNEL_DTYPES and weight.dtype == x.dtype
            and weight.device == x.device and weight.dim() == 1 and x.shape[-1] <= MAX_FEATURES
            and type(x) in _PLAIN and type(weight) in _PLAIN and not torch.is_autocast_enabled('cuda')
            and not torch._C._are_functorch_transforms_active() and torch.autograd.forward_ad._current_level < 0
            and not torch.compiler.is_compiling() and _lib.nodes_available())


def _rms(x, weight, eps):
    if x.is_cuda and weight is not None and weight.numel() == x.shape[-1]:
        if eps is not None and _trains_on_kernels(x, weight):  # (torch's op takes the type's own then)
            return rms_norm_rows(x, weight, eps)
        return F.rms_norm(x, (x.shape[-1],), weight, eps)
    x_f = x.float()
    y = (x_f * torch.rsqrt(x_f.pow(2).mean(-1, keepdim=True) + eps)).to(x.dtype)
    return y * weight if weight is not None else y


class RMSNorm(nn.Module):
    '''Root-mean-square normalisation over the last dimension.'''

    def __init__(self, dim, eps=1e-6, elementwise_affine=True, use_triton=True):
        super().__init__()
        self.dim = dim
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        if elementwise_affine:
            self.weight = nn.Parameter(torch.ones(dim))
        else:
            self.register_parameter('weight', None)
        self.use_triton = False

    def forward(self, x):
        return _rms(x, self.weight, self.eps)


class GatedRMSNorm(nn.Module):
    '''RMSNorm of the value half of [values || gate], gated by SiLU(gate).'''

    def __init__(self, dim, eps=1e-6, elementwise_affine=True, use_triton=True):
        super().__init__()
        self.dim = dim
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        if elementwise_affine:
            self.weight = nn.Parameter(torch.ones(dim))
        else:
            self.register_parameter('weight', None)
        self.use_triton = False

    def forward(self, x):
        x_in, gate = x.split(self.dim, dim=-1)
        x_f = x_in.float()
        y = (x_f * torch.rsqrt(x_f.pow(2).mean(-1, keepdim=True) + self.eps)).to(x.dtype)
        if self.weight is not None:
            y = y * self.weight
        return y * F.silu(gate)
