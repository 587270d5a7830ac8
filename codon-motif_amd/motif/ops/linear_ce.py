'''Softmax cross entropy straight from hidden states, the logits never stored
(csrc/linear_ce.hip; the reference forms the logits and calls F.cross_entropy on them,
motif/model/motif.py:600-628).
'''
import torch

from . import _lib
from .autograd_path import refuse_transforms

MAX_ROWS, MAX_FEATURES, MAX_VOCABULARY = 2 ** 23, 2 ** 16, 2 ** 22 - 64
_REDUCTIONS = {'none': 0, 'sum': 1, 'mean': 2}


def _row_major(t):
    '''t, or a copy, with features beside each other and rows that do not overlap.'''
    return t if t.stride(1) == 1 and (t.shape[0] < 2 or t.stride(0) >= t.shape[1]) else t.contiguous()


def linear_cross_entropy(x, weight, labels, ignore_index=-100, reduction='mean'):
    '''F.cross_entropy(F.linear(x, weight).float(), labels, ignore_index=, reduction=) without the
    logits in memory: x [..., d] hidden states, weight [V, d] of the same dtype (bf16 or
    fp32), labels [...] int64.  Returns fp32: a scalar, or one loss per label for 'none' (0
    where ignored).  The mean is over the labels that count (NaN when none does).

    Rows whose label is `ignore_index` are left out of every product: they get a zero
    gradient and nothing that they hold reaches the loss.  A label outside [0, V) that is not
    `ignore_index` gives NaN (loss and gradients).  Under autocast, x and weight are cast to its
    dtype, as F.linear does.  Differentiable once in x and weight, in reverse mode; tracing,
    function transforms and forward-mode tangents are refused.

    For the backward a copy of the labelled rows, the weight and 16 bytes a row are kept.  Its scratch
    is the gradient of the logits in pieces of the vocabulary (256 MB to 1 GB, or 4096 vocabulary
    rows where that is more; for all rows, labelled or not), and partial sums of x's gradient in
    fp32.  The forward's is two fp32 numbers for each row and 128 (bf16) or 32 (fp32) vocabulary rows.

    In bf16 the logits' gradient is rounded to bf16 for its products, but for steps of up to 32 labelled rows.'''
    refuse_transforms('linear_cross_entropy', x, weight, labels)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f'linear_cross_entropy: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match')
    if labels.shape != x.shape[:-1]:
        raise ValueError(f'linear_cross_entropy: labels {tuple(labels.shape)} for x {tuple(x.shape)}')
    if labels.dtype not in (torch.int64, torch.int32):
        raise ValueError(f'linear_cross_entropy: labels must be int64, got {labels.dtype}')
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f'linear_cross_entropy: an empty weight {tuple(weight.shape)}')
    if weight.device != x.device or labels.device != x.device:
        raise ValueError(f'linear_cross_entropy: x on {x.device}, weight on {weight.device}, labels on {labels.device}')
    if torch.is_autocast_enabled(x.device.type):
        dt = torch.get_autocast_dtype(x.device.type)
        x, weight = x.to(dt), weight.to(dt)
    if x.dtype != weight.dtype:
        raise ValueError(f'linear_cross_entropy: x is {x.dtype}, weight {weight.dtype}')
    _lib.dtype_code(x.dtype)
    N, d = labels.numel(), x.shape[-1]
    if N > MAX_ROWS or weight.shape[0] > MAX_VOCABULARY or d > MAX_FEATURES:
        raise ValueError(f'linear_cross_entropy: {N} rows of {d} features over {weight.shape[0]} are out of range')
    if not x.is_cuda:
        raise ValueError(f'linear_cross_entropy: x is on {x.device}, the kernels need a ROCm device')
    if N == 0:  # (connected to the graph; the sum of nothing, and its mean)
        zero = x.float().sum() + 0.0 * weight[:0].float().sum()
        return {'none': zero.expand(labels.shape), 'sum': zero, 'mean': zero * float('nan')}[reduction]
    red = _REDUCTIONS[reduction]
    x2, lab = x.reshape(-1, d), labels.reshape(-1).to(torch.int64)
    x2 = x2 if x2.stride(1) == 1 else x2.contiguous()
    loss = _lib.nodes().linear_ce(x2, _row_major(weight), lab, int(ignore_index), red)
    return loss.view(labels.shape) if red == 0 else loss
