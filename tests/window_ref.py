'''Chord attention under a window in float64, with the largest distance from it that the
kernels' roundings allow, and the values of 4-bit rows.'''
import math

import torch

from support import gen


def inputs(B, H, Hkv, L, S, D, dtype, seed=0, mu_scale=1.0):
    '''q, k, v, (alpha, beta, mu, ssmax) on the CPU: unit-size rows, parameters of the
    size a trained layer has.'''
    g = gen(seed)
    q, k = torch.randn(B, H, L, D, generator=g), torch.randn(B, Hkv, S, D, generator=g)
    v = 0.5 * torch.randn(B, Hkv, S, D, generator=g)
    par = (torch.exp(0.3 * torch.randn(H, generator=g)), 0.2 * torch.randn(H, generator=g),
           mu_scale * 0.2 * torch.randn(H, generator=g), 1 + 0.1 * torch.randn(H, generator=g))
    return q.to(dtype), k.to(dtype), v.to(dtype), par


def log_n_of(B, L, q_start):
    return torch.log(torch.arange(q_start + 1, q_start + L + 1, dtype=torch.float32))[None].expand(B, L).contiguous()


def seen(L, S, q_start, window, sinks):
    i = q_start + torch.arange(L)[:, None]
    j = torch.arange(S)[None]
    keep = j <= i
    if window is not None:
        keep = keep & ((j > i - window) | (j < sinks))
    return keep


def attention64(q, k, v, par, log_n, q_start, window=None, sinks=0, scale=None, eps=1e-5):
    '''(out, lse in log2 units, allowed): `allowed` bounds |kernel - out| elementwise.

    With u = 2^-24 and p the softmax weights: a logit z = c (s q.k + b) is off by at most
      dz = |c| (s (D + 4) u sum|q k| + 2^-19 |b|) + 8 u |z|
    (fp32 sums of D terms; the bias through log2 and exp2, each within 2^-23 of arguments up
    to 13), a weight by 2 max dz + 2^-21 relative, the sum over keys by 64 u (pairwise or
    short chains).  16-bit outputs add a weight's rounding to that type, h = eps / 2 of it
    (the sums run in fp32), and the output's own.'''
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    par = [t.detach().cpu().double() for t in par]
    log_n = log_n.detach().cpu().double()
    B, H, L, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    k, v = (t.repeat_interleave(H // Hkv, 1) for t in (k, v))
    al, be, mu, ss = (t.view(H, 1, 1) for t in par)
    d = (torch.arange(S)[None] - (q_start + torch.arange(L)[:, None])).double()
    b = -al * ((d - mu).abs() + eps) ** be
    c = ss * log_n[:, None, :, None]
    u = 2.0 ** -24
    z = c * (scale * (q @ k.transpose(-1, -2)) + b)
    dz = c.abs() * (abs(scale) * (D + 4) * u * (q.abs() @ k.abs().transpose(-1, -2)) + 2.0 ** -19 * b.abs()) + 8 * u * z.abs()
    keep = seen(L, S, q_start, window, sinks)
    p = torch.softmax(z.masked_fill(~keep, -1e300), -1) * keep
    out = p @ v
    lse = torch.logsumexp(z.masked_fill(~keep, -math.inf), -1) / math.log(2)
    worst = (dz * keep).amax(-1, keepdim=True)
    return out, lse, (2 * worst + 2.0 ** -21 + 64 * u) * (p @ v.abs())


def assert_near(got, out, allowed, v_abs_mean, dtype, what=''):
    '''`allowed` plus the roundings of a 16-bit type: the weights' (h times the mean of |v|
    under the weights) and the output's (h of it, and half the smallest subnormal).'''
    h = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    lim = allowed + h * v_abs_mean + (h + 2.0 ** -23) * out.abs() + 2.0 ** -25
    d = (got.detach().cpu().double() - out).abs()
    bad = ~(d <= lim)  # (NaN is bad)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / lim).max()):.2f} of the limit'


def check_attention(got, q, k, v, par, log_n, q_start, window=None, sinks=0, scale=None, what='', rounded=None):
    '''`rounded` (default |v|): the sizes that a weight's rounding to a 16-bit type multiplies.'''
    dt = q.dtype
    out, _, allowed = attention64(q, k, v, par, log_n, q_start, window, sinks, scale)
    rounded = (v if rounded is None else rounded).detach().cpu().double().abs()
    mean, _, _ = attention64(q, k, rounded, par, log_n, q_start, window, sinks, scale)
    assert_near(got, out, allowed, mean, dt, what)


def quantise64(x):
    '''(codes [.., D], scale, base [.., groups]) of rows x: the range in fp32, scale and base
    held in bf16, the quotient in fp32, as the format defines them.'''
    grp = min(32, x.shape[-1])
    g = x.detach().cpu().float().unflatten(-1, (-1, grp))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) * torch.tensor(1 / 15, dtype=torch.float32)).bfloat16()
    base = lo.bfloat16()
    q = (g - base.float()[..., None]) / scale.float()[..., None]
    code = torch.where(scale[..., None] == 0, torch.zeros_like(q), q.round().clamp(0, 15))
    return code.flatten(-2), scale, base


def values64(codes, scale, base):
    g = codes.double().unflatten(-1, (scale.shape[-1], -1))
    return (g * scale.double()[..., None] + base.double()[..., None]).flatten(-2)


def slab_values64(slab):
    '''(k, v) float64 on the CPU of every position of a KV4Slab.'''
    out = []
    for c, p in ((slab.k_codes, slab.k_params), (slab.v_codes, slab.v_params)):
        c, p = c.cpu(), p.cpu()
        codes = torch.stack([c & 15, c >> 4], -1).flatten(-2)
        out.append(values64(codes, p[..., 0], p[..., 1]))
    return out


def code_sizes64(slab):
    '''max(|v|, scale |code - 8|) of every value of a KV4Slab: over 4-bit rows the product with the
    weights runs on v = scale (code - 8) + (base + 8 scale), the weight p scale rounded to the
    matrix instructions' type and multiplied by code - 8, the rest in fp32; so a weight's
    rounding h moves the output by h p scale |code - 8|, where expanded values would give h p |v|.'''
    c, p = slab.v_codes.cpu(), slab.v_params.cpu()
    codes = torch.stack([c & 15, c >> 4], -1).flatten(-2)
    scale = p[..., 0].double().abs()
    off = (codes.double() - 8).abs().unflatten(-1, (scale.shape[-1], -1)) * scale[..., None]
    return torch.maximum(values64(codes, p[..., 0], p[..., 1]).abs(), off.flatten(-2))


def random_slab(B, Hkv, cap, D, device, seed=0):
    '''A slab of rows quantised in torch (independent of the kernels): unit-size keys, values
    of half size with an offset.'''
    from motif.ops import KV4Slab
    g = gen(seed)
    ts = []
    for off, size in ((0.0, 1.0), (0.3, 0.5)):
        x = off + size * torch.randn(B, Hkv, cap, D, generator=g)
        code, scale, base = quantise64(x)
        code = code.to(torch.uint8)
        ts += [code[..., 0::2] | (code[..., 1::2] << 4), torch.stack([scale, base], -1)]
    return KV4Slab(*[t.contiguous().to(device) for t in ts])


def over_rows64(q, rows, k, v, par, log_n, q_start, window, sinks, eps=1e-5):
    '''(out, the same of |v|) in float64 where only the keys at positions `rows` (given as k, v) count.'''
    H, L, D = q.shape[1:]
    al, be, mu, ss = (t.double().view(H, 1, 1) for t in par)
    pos = torch.tensor(rows, dtype=torch.float64)
    G = H // k.shape[1]
    k, v = (t.cpu().double().repeat_interleave(G, 1) for t in (k, v))
    i = (q_start + torch.arange(L))[:, None].double()
    d = pos[None] - i
    z = (q.double() @ k.transpose(-1, -2) * D ** -0.5 - al * ((d - mu).abs() + eps) ** be) * (ss * log_n.double()[:, None, :, None])
    z = z.masked_fill(~((d <= 0) & ((d > -window) | (pos < sinks)[None])), float('-inf'))
    p = torch.softmax(z, -1)
    return p @ v, p @ v.abs()
