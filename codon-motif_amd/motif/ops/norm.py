'''RMSNorm and LayerNorm of rows with their gradients (csrc/row_norm.hip).

The forward of the reference's row norms (motif/ops/rms_norm.py:17-61) in one pass over
fp32 arithmetic, rounded once, and their backward (:63-112) with the weight's gradient
summed in a fixed order.  `RMSNorm` calls `rms_norm_rows` where gradients are wanted.
'''
import torch

from . import _lib
from .autograd_path import wants_grad

MAX_FEATURES = 16384


def _rows(t):
    '''t as [rows, D] with features beside each other: a view where its strides allow one.'''
    if t.dim() == 2 and t.stride(1) == 1:
        return t
    D = t.shape[-1]
    if t.stride(-1) != 1:
        t = t.contiguous()
    return t.reshape(-1, D)


def _launch(x2, weight, bias, y2, stats, eps, layer):
    rows, D = x2.shape
    dev = x2.device
    rstd = mean = None
    if stats is not None:
        rstd = stats.data_ptr()
        mean = rstd + 4 * rows if layer else None
    with _lib.on_device(dev):
        rc = _lib.lib().motif_row_norm_fwd(
            x2.data_ptr(), x2.stride(0), _lib.ptr(weight), _lib.ptr(bias), y2.data_ptr(), y2.stride(0), rstd, mean,
            rows, D, eps, layer, _lib.chord_dtype_code(x2.dtype), _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, 'motif_row_norm_fwd')


def _norm_torch(x, weight, bias, eps, layer):
    '''The same in torch ops, for derivatives beyond the first.'''
    h = x.float()
    if layer:
        h = h - h.mean(-1, keepdim=True)
    h = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps)
    if weight is not None:
        h = h * weight.float()
    if bias is not None:
        h = h + bias.float()
    return h.to(x.dtype)


class RowNormFunction(torch.autograd.Function):
    '''motif_row_norm_fwd / motif_row_norm_bwd: gradients for x, weight and bias (their own derivatives, where
    a graph of them is asked for, through torch ops).'''

    @staticmethod
    def forward(ctx, x, weight, bias, eps, layer):
        x2 = _rows(x)
        rows, D = x2.shape
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = torch.empty((2 if layer else 1) * rows, dtype=torch.float32, device=x.device)
        if rows:
            _launch(x2, weight, bias, y.view(rows, D), stats, eps, layer)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.layer, ctx.eps = layer, eps
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        layer = ctx.layer
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        if torch.is_grad_enabled():  # (create_graph: what the kernels give carries no graph)
            leaves = [t for t, need in zip((x, weight, bias), ctx.needs_input_grad) if need]
            got = iter(torch.autograd.grad(_norm_torch(x, weight, bias, ctx.eps, layer), leaves, dy, create_graph=True))
            return next(got) if need_x else None, next(got) if need_w else None, next(got) if need_b else None, None, None
        x2, dy2 = _rows(x), _rows(dy)
        rows, D = x2.shape
        dev, dt = x.device, x.dtype
        dx = torch.empty(x.shape, dtype=dt, device=dev) if need_x else None
        dw = torch.empty(D, dtype=dt, device=dev) if need_w else None
        db = torch.empty(D, dtype=dt, device=dev) if need_b else None
        if rows == 0:
            return dx, (dw.zero_() if need_w else None), (db.zero_() if need_b else None), None, None
        lib = _lib.lib()
        ws, nbytes = None, 0
        if need_w or need_b:
            nbytes = lib.motif_row_norm_bwd_workspace_bytes(rows, D, layer)
            ws = torch.empty(nbytes // 4, dtype=torch.float32, device=dev)
        rstd = stats.data_ptr()
        with _lib.on_device(dev):
            rc = lib.motif_row_norm_bwd(
                dy2.data_ptr(), dy2.stride(0), x2.data_ptr(), x2.stride(0), _lib.ptr(weight), rstd,
                rstd + 4 * rows if layer else None, _lib.ptr(dx), D, _lib.ptr(dw), _lib.ptr(db), rows, D, layer,
                _lib.ptr(ws), nbytes, _lib.chord_dtype_code(dt), _lib.stream_ptr(dev))
        if rc:
            _lib.check(rc, 'motif_row_norm_bwd')
        return dx, dw, db, None, None


def _check(x, params, what):
    if x.dtype not in (torch.bfloat16, torch.float16, torch.float32):
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
        if tuple(t.shape) != (D,) or t.dtype != x.dtype or t.device != x.device:
            raise ValueError(f'{what}: {name} must be [{D}] of {x.dtype} on {x.device}, got {tuple(t.shape)} of '
                             f'{t.dtype} on {t.device}')
    if not x.is_cuda:
        raise ValueError(f'{what}: x is on {x.device}, the kernels need a ROCm device')


def _norm(x, weight, bias, eps, layer, what):
    _check(x, (('weight', weight), ('bias', bias)), what)
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if wants_grad(x, weight, bias):
        return RowNormFunction.apply(x, weight, bias, float(eps), layer)
    x2 = _rows(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if x2.shape[0]:
        _launch(x2, weight, bias, y.view(x2.shape), None, float(eps), layer)
    return y


def rms_norm_rows(x, weight=None, eps=1e-6):
    '''x / sqrt(mean(x^2) + eps) * weight over the last dimension of x [..., D] (fp32, bf16 or
    fp16, D at most 16384), in fp32, rounded once.  weight [D] of x's dtype, or None.
    Differentiable in x and weight.'''
    return _norm(x, weight, None, eps, 0, 'rms_norm_rows')


def layer_norm_rows(x, weight=None, bias=None, eps=1e-5):
    '''(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of x [..., D], as
    rms_norm_rows; bias [D] of x's dtype, or None.  Differentiable in x, weight and bias.'''
    return _norm(x, weight, bias, eps, 1, 'layer_norm_rows')
