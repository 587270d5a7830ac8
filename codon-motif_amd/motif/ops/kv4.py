'''A key / value cache held in 4 bits, and Chord attention over it, on the gfx950 HIP
kernels (new; the reference keeps its caches in the activation type).

For every (batch row, kv head, position), keys and values alike, a `KV4Slab` holds

  codes   uint8 [B, Hkv, capacity, D / 2]: feature 2 m of the row in the low half of byte
          m, feature 2 m + 1 in the high half;
  params  bfloat16 [B, Hkv, capacity, D / min(32, D), 2]: (scale, base) of every group of
          min(32, D) features; a feature's value is code * scale + base.

`kv4_append` writes rows (base = bf16(min), scale = bf16((max - min) / 15), the code
nearest to (x - base) / scale, ties to even), `kv4_read` gives the values back,
`chord_kv4_prep` writes a decode step's rows straight from its projections, and
`chord_attention_kv4` / `chord_decode_kv4_cursor` attend over the cache without
expanding it in memory: 40 bytes a row at head dim 64 where bf16 takes 128.  All of them
are forward-only: calls that would need a gradient raise.
'''
import functools
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .autograd_path import wants_grad
from .chord_attention import _DTYPES, HEAD_DIMS, NO_WINDOW, _check_params, _out_for, _rows4, check_window

GROUP = 32  # features that share a (scale, base) pair


class KV4Slab(NamedTuple):
    '''The four tensors of a 4-bit cache (positions back to back, any batch / head strides; one whose
    batch rows or heads share memory, an expanded one, is for reading only).'''
    k_codes: torch.Tensor
    k_params: torch.Tensor
    v_codes: torch.Tensor
    v_params: torch.Tensor

    @property
    def capacity(self) -> int:
        return self.k_codes.shape[2]

    @property
    def head_dim(self) -> int:
        return 2 * self.k_codes.shape[3]


def kv4_alloc(batch: int, kv_heads: int, capacity: int, head_dim: int, device) -> KV4Slab:
    '''A zeroed slab (every value 0) of `capacity` positions.'''
    if head_dim not in HEAD_DIMS:
        raise ValueError(f'kv4_alloc: head_dim must be one of {HEAD_DIMS}, got {head_dim}')
    codes = (batch, kv_heads, capacity, head_dim // 2)
    params = (batch, kv_heads, capacity, head_dim // min(GROUP, head_dim), 2)
    z = lambda s, dt: torch.zeros(s, dtype=dt, device=device)
    return KV4Slab(z(codes, torch.uint8), z(params, torch.bfloat16), z(codes, torch.uint8), z(params, torch.bfloat16))


def _check_slab(slab: KV4Slab, what: str, writes: bool = False):
    '''((B, Hkv, capacity, D), the entry points' arguments), or ValueError.'''
    kc, kp, vc, vp = slab
    shape = kc.shape
    if len(shape) != 4 or kc.dtype != torch.uint8 or vc.dtype != torch.uint8:
        raise ValueError(f'{what}: codes must be uint8 [B, Hkv, capacity, D / 2]')
    B, Hkv, cap, half = shape
    D = 2 * half
    if D not in HEAD_DIMS:
        raise ValueError(f'{what}: head_dim must be one of {HEAD_DIMS}, got {D}')
    G = D // GROUP if D > GROUP else 1
    pshape = (B, Hkv, cap, G, 2)
    if vc.shape != shape or kp.shape != pshape or vp.shape != pshape \
            or kp.dtype != torch.bfloat16 or vp.dtype != torch.bfloat16:
        raise ValueError(f'{what}: codes of keys and values must have one shape, params must be bfloat16 {pshape}')
    args = []
    for c, p in ((kc, kp), (vc, vp)):
        cs, ps, cp, pp = c.stride(), p.stride(), c.data_ptr(), p.data_ptr()
        if B and Hkv and cap:
            if cs[3] != 1 or (cap > 1 and cs[2] != half) or (cp | cs[0] | cs[1]) & 3:
                raise ValueError(f'{what}: rows of codes must lie back to back on 4-byte boundaries')
            if ps[4] != 1 or (G > 1 and ps[3] != 2) or (cap > 1 and ps[2] != 2 * G) or pp & 3 or (ps[0] | ps[1]) & 1:
                raise ValueError(f'{what}: rows of params must lie back to back on 4-byte boundaries')
        if writes and (B > 1 and not (cs[0] and ps[0]) or Hkv > 1 and not (cs[1] and ps[1])):
            raise ValueError(f'{what}: the rows or heads of the cache share memory')
        args += (cp, cs[0], cs[1], pp, ps[0] >> 1, ps[1] >> 1)
    at = kc.get_device()
    if at < 0:
        raise ValueError(f'{what}: the cache must live on CUDA')
    if kp.get_device() != at or vc.get_device() != at or vp.get_device() != at:
        raise ValueError(f'{what}: the cache tensors must live on one device')
    return (B, Hkv, cap, D), args


def _need_backend():
    if not _lib.available():
        raise RuntimeError('there is no usable HIP backend in the current environment')


def kv4_append(slab: KV4Slab, k: torch.Tensor, v: torch.Tensor, start) -> None:
    '''Write the rows k, v [B, Hkv, n, D] (fp16, bf16 or fp32, any strides) at positions
    [start, start + n) of the slab.  `start` is an int, or a device int32 tensor of one
    entry that the kernel reads (for a captured step; rows past the capacity are then
    dropped).  A group of features that holds an infinity or a NaN, or whose
    range passes fp32's largest number, reads back as NaN; fp32 features past bf16's
    largest (3.3895e38) count as that.'''
    if wants_grad(k, v):
        raise RuntimeError('kv4_append is forward-only: detach the rows or call it under no_grad')
    (B, Hkv, cap, D), args = _check_slab(slab, 'kv4_append', writes=True)
    if k.shape != v.shape or k.dim() != 4 or k.shape[:2] != (B, Hkv) or k.shape[3] != D:
        raise ValueError(f'kv4_append: k / v must be [{B}, {Hkv}, n, {D}], got {tuple(k.shape)} and {tuple(v.shape)}')
    if k.dtype != v.dtype or k.device != slab.k_codes.device or v.device != k.device:
        raise ValueError('kv4_append: k, v and the cache must share a device, k and v a dtype')
    n = k.shape[2]
    if isinstance(start, torch.Tensor):
        if start.dtype != torch.int32 or start.device != k.device or start.numel() != 1:
            raise ValueError('kv4_append: a tensor `start` must be one int32 on the cache\'s device')
        dev, pos = start.data_ptr(), 0
    else:
        dev, pos = None, int(start)
        if pos < 0 or pos + n > cap:
            raise ValueError(f'kv4_append: positions [{pos}, {pos + n}) outside a cache of {cap}')
    _need_backend()
    if k.numel() == 0:
        return
    k4, v4 = _rows4(k), _rows4(v)
    with _lib.on_device(k.device):
        rc = _lib.lib().motif_kv4_append(*k4[1], *v4[1], *args, dev, pos, cap, B, n, Hkv, D,
                                         _lib.chord_dtype_code(k.dtype), _lib.stream_ptr(k.device))
    if rc:
        _lib.check(rc, 'motif_kv4_append')


def kv4_read(slab: KV4Slab, start: int, n: int, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    '''The values of positions [start, start + n) as (k, v), new [B, Hkv, n, D] tensors of
    `dtype` (fp16, bf16 or fp32; the fp32 value rounded once, in fp16 held at +-65504 where
    rounding would give an infinity).'''
    (B, Hkv, cap, D), args = _check_slab(slab, 'kv4_read')
    start, n = int(start), int(n)
    if start < 0 or n < 0 or start + n > cap:
        raise ValueError(f'kv4_read: positions [{start}, {start + n}) outside a cache of {cap}')
    code = _lib.chord_dtype_code(dtype)
    _need_backend()
    k = torch.empty(B, Hkv, n, D, dtype=dtype, device=slab.k_codes.device)
    v = torch.empty_like(k)
    if k.numel():
        s0, s1, s2, _ = k.stride()
        with _lib.on_device(k.device):
            rc = _lib.lib().motif_kv4_read(*args, k.data_ptr(), s0, s1, s2, v.data_ptr(), s0, s1, s2, start, cap, B, n, Hkv,
                                           D, code, _lib.stream_ptr(k.device))
        if rc:
            _lib.check(rc, 'motif_kv4_read')
    return k, v


def chord_kv4_prep(proj: torch.Tensor, offsets, q_norm_weight: torch.Tensor, k_norm_weight: torch.Tensor, norm_eps: float,
                   slab: KV4Slab, length_dev: torch.Tensor, num_heads: int) -> torch.Tensor:
    '''The input side of a Chord decode step over a 4-bit cache in one launch: from the fused
    projection rows proj [B, L, ncols] (bf16 or fp32; q, k, v from column offsets[i]), q [B, H, L, D]
    normalised, and the normalised keys and the values written in 4 bits at positions length_dev ..
    (a device int32, read and not advanced; rows past the capacity are dropped).  The same bits as the
    norms followed by kv4_append.'''
    (B, Hkv, cap, D), args = _check_slab(slab, 'chord_kv4_prep', writes=True)
    if wants_grad(proj, q_norm_weight, k_norm_weight):
        raise RuntimeError('chord_kv4_prep is forward-only: call it under no_grad')
    if proj.dim() != 3 or proj.shape[0] != B or proj.stride(-1) != 1 or proj.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f'chord_kv4_prep: proj must be bf16 or fp32 [{B}, L, columns], got {tuple(proj.shape)} {proj.dtype}')
    offsets = [int(o) for o in offsets]
    if num_heads < 1 or num_heads % Hkv or len(offsets) != 3 or min(offsets) < 0 \
            or max(offsets[0] + num_heads * D, max(offsets[1:]) + Hkv * D) > proj.shape[2]:
        raise ValueError(f'chord_kv4_prep: {num_heads} heads of {D} over {Hkv} kv heads do not fit the columns {offsets}')
    for t in (q_norm_weight, k_norm_weight):
        if t.shape != (D,) or t.dtype != proj.dtype or not t.is_contiguous() or t.device != proj.device:
            raise ValueError(f'chord_kv4_prep: norm weights must be contiguous [{D}] in proj\'s dtype and on its device')
    if slab.k_codes.device != proj.device:
        raise ValueError('chord_kv4_prep: proj and the cache must live on one device')
    if length_dev.dtype != torch.int32 or length_dev.device != proj.device or length_dev.numel() != 1:
        raise ValueError('chord_kv4_prep: length_dev must be one int32 on proj\'s device')
    _need_backend()
    q = torch.empty(B, num_heads, proj.shape[1], D, dtype=proj.dtype, device=proj.device)
    if q.numel() == 0:
        return q
    with _lib.on_device(proj.device):
        rc = _lib.lib().motif_chord_kv4_prep(
            proj.data_ptr(), proj.stride(0), proj.stride(1), *offsets, q_norm_weight.data_ptr(), k_norm_weight.data_ptr(),
            float(norm_eps), *_lib.t4(q), *args, length_dev.data_ptr(), cap, B, proj.shape[1], num_heads, Hkv, D,
            _lib.dtype_code(proj.dtype), _lib.stream_ptr(proj.device))
    _lib.check(rc, 'motif_chord_kv4_prep')
    return q


def _check_query(q, slab, params, what):
    (B, Hkv, cap, D), args = _check_slab(slab, what)
    shape, at = q.shape, q.get_device()
    if len(shape) != 4 or shape[0] != B or shape[3] != D or shape[1] % Hkv:
        raise ValueError(f'{what}: q {tuple(shape)} does not fit a cache of {B} rows, {Hkv} kv heads of {D}')
    if q.dtype not in _DTYPES or q.stride()[3] != 1:
        raise ValueError(f'{what}: q must be fp16 / bf16 / fp32 and contiguous along the last dimension')
    if at != slab[0].get_device():
        raise ValueError(f'{what}: q and the cache must live on one device')
    _check_params(*params, shape[1])
    for t in params:
        if t.get_device() != at:
            raise ValueError(f'{what}: the head parameters must live on q\'s device')
    return B, shape[1], Hkv, shape[2], D, cap, args


def _launch_kv4(q, args, Hkv, params, log_n, log_table, length_dev, S, q_start, scale, eps, window, sinks, out, workspace):
    B, H, L, D = q.shape
    q, q4 = _rows4(q)
    code = _lib.chord_dtype_code(q.dtype)
    dev = q.device
    with _lib.on_device(dev):
        if workspace is None:
            n = _kv4_workspace_bytes(B, H, Hkv, L, S, D, window, sinks, code)
            workspace = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        alpha, beta, mu, ssmax = params
        rc = _lib.lib().motif_chord_kv4_fwd(
            *q4, *args, alpha.data_ptr(), beta.data_ptr(), mu.data_ptr(), ssmax.data_ptr(),
            *((None, 0, 0) if log_n is None else (log_n.data_ptr(), *log_n.stride())),
            *((None, 0) if log_table is None else (log_table.data_ptr(), log_table.numel())),
            out.data_ptr(), *out.stride()[:3], None if length_dev is None else length_dev.data_ptr(),
            B, H, Hkv, L, S, D, q_start, scale, eps, window, sinks,
            None if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.numel(), code,
            _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, 'motif_chord_kv4_fwd')
    return out


@functools.lru_cache(maxsize=256)
def _kv4_workspace_bytes(*sizes) -> int:
    return int(_lib.lib().motif_chord_kv4_workspace_bytes(*sizes))


def chord_attention_kv4(q: torch.Tensor, slab: KV4Slab, alpha, beta, mu, ssmax, log_n: torch.Tensor, length: int,
                        softmax_scale: Optional[float] = None, eps: float = 1e-5,
                        window: Optional[int] = None, sinks: int = 0,
                        out: Optional[torch.Tensor] = None) -> torch.Tensor:
    '''Chord attention of the last L of `length` positions over the first `length` rows of
    a 4-bit cache: apply_chord_attention of the values that the rows stand for.

    q [B, H, L, D] (fp16, bf16 or fp32), alpha .. ssmax [H] fp32, log_n [B, L] fp32,
    `window` / `sinks` and `out` as for apply_chord_attention.  Returns [B, H, L, D] in
    q's dtype.  Forward-only.'''
    if wants_grad(q, alpha, beta, mu, ssmax, log_n):
        raise RuntimeError('chord_attention_kv4 is forward-only: call it under no_grad')
    window, sinks = check_window(window, sinks)
    params = (alpha, beta, mu, ssmax)
    B, H, Hkv, L, D, cap, args = _check_query(q, slab, params, 'chord_attention_kv4')
    length = int(length)
    if not L <= length <= cap:
        raise ValueError(f'chord_attention_kv4: length {length} must lie between the {L} queries and the capacity {cap}')
    if log_n.shape != (B, L) or log_n.dtype != torch.float32 or log_n.device != q.device:
        raise ValueError(f'log_n must be fp32 [{B}, {L}] on q\'s device')
    _need_backend()
    out = _out_for(out, q)
    if out.numel() == 0:
        return out
    return _launch_kv4(q, args, Hkv, params, log_n, None, None, length, length - L,
                       D ** -0.5 if softmax_scale is None else float(softmax_scale), float(eps),
                       NO_WINDOW if window is None else window, sinks, out, None)


def chord_decode_kv4_workspace(B, H, Hkv, L, capacity, D, dtype, device, window=None, sinks=0) -> Optional[torch.Tensor]:
    '''A workspace for chord_decode_kv4_cursor at these sizes (None where it needs none).'''
    window, sinks = check_window(window, sinks)
    n = _kv4_workspace_bytes(B, H, Hkv, L, capacity, D, NO_WINDOW if window is None else window, sinks,
                             _lib.chord_dtype_code(dtype))
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def chord_decode_kv4_cursor(q, slab: KV4Slab, length_dev, alpha, beta, mu, ssmax, log_table, softmax_scale=None,
                            eps=1e-5, window=None, sinks=0, workspace=None):
    '''chord_attention_kv4 at the device cursor: `length_dev` (device int32) positions are
    cached and the L new rows lie behind them (kv4_append with start=length_dev puts them
    there).  Attends with q_start = length_dev and log_n[b, i] = log_table[q_start + i],
    then advances length_dev by L on the device, so a captured step replays token after
    token.  Two launches that may run at once must not share `workspace`.'''
    if wants_grad(q, alpha, beta, mu, ssmax):
        raise RuntimeError('chord_decode_kv4_cursor is forward-only: call it under no_grad')
    window, sinks = check_window(window, sinks)
    params = (alpha, beta, mu, ssmax)
    B, H, Hkv, L, D, cap, args = _check_query(q, slab, params, 'chord_decode_kv4_cursor')
    if length_dev.dtype != torch.int32 or length_dev.device != q.device or length_dev.numel() != 1:
        raise ValueError('chord_decode_kv4_cursor: length_dev must be one int32 on q\'s device')
    if log_table.dtype != torch.float32 or log_table.device != q.device or log_table.numel() < cap \
            or not log_table.is_contiguous():
        raise ValueError('chord_decode_kv4_cursor: log_table must be contiguous fp32 with at least `capacity` entries')
    if L > cap:
        raise ValueError('chord_decode_kv4_cursor: more queries than the capacity')
    _need_backend()
    out = _out_for(None, q)
    if out.numel() == 0:
        return out
    return _launch_kv4(q, args, Hkv, params, None, log_table, length_dev, cap, 0,
                       D ** -0.5 if softmax_scale is None else float(softmax_scale), float(eps),
                       NO_WINDOW if window is None else window, sinks, out, workspace)
