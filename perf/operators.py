'''Chord attention with a sliding window and visible first tokens, and over a 4-bit cache:
the calls that a program makes of these operators, for timing and comparison.

  window_prefill  apply_chord_attention(window=, sinks=) over a prompt or a later piece of one
  window_train    the same op forward and backward
  window_decode   the same op, one or two new tokens over a cached context
  kv4_write       kv4_append of new rows to a 4-bit cache and kv4_read of them back
  kv4_decode      chord_attention_kv4: new tokens over a context held in 4 bits

A query at position p sees key j when j <= p and (j > p - window or j < sinks).

A 4-bit cache holds, for every (batch row, kv head, position), D codes of 4 bits (byte m:
feature 2 m in the low half, 2 m + 1 in the high half) and, for every group of min(32, D)
features, a bf16 pair (scale, base): value = code * scale + base, with
  scale = bf16((max - min) * fp32(1 / 15)), base = bf16(min) over the group,
  code = (value - base) / scale in fp32, rounded to even and clamped to 0 .. 15 (0 where
  the scale is 0).

Sizes: 12 heads, 3 kv heads of 64, 2048 and 4096 tokens, a context of 4097 and 64 decode
rows are the 172M model's and the benchmark's; the rest are generic.
'''
import math
import os
import sys

import torch

own = False

DEV = 'cuda'
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
NORM_EPS = 1e-6  # of the q / k norms in front of the op
GGD_EPS = 1e-5   # of the distance bias
GROUP = 32       # features that share a scale


def listed():
    return [
        # the attention op of a 4096-token prompt at the model's grouped heads, local layers
        dict(name='window_prefill_bf16_t4096', kind='window_prefill', dtype='bf16', B=1, H=12, Hkv=3, D=64, L=4096,
             S=4096, window=1024, sinks=4),
        # a long prompt, a wide window: the largest pass
        dict(name='window_prefill_bf16_t8192', kind='window_prefill', dtype='bf16', B=1, H=12, Hkv=3, D=64, L=8192,
             S=8192, window=2048, sinks=16),
        # a ragged later piece of two prompts in the accuracy mode, an odd window, no first tokens
        dict(name='window_prefill_fp32_t517', kind='window_prefill', dtype='fp32', B=2, H=12, Hkv=3, D=64, L=517,
             S=1023, window=259, sinks=0),
        # a training step's share of one layer, two sequences, as many kv heads as heads
        dict(name='window_train_b2_t2048', kind='window_train', B=2, H=12, Hkv=12, L=2048, window=512, sinks=4),
        # the same on one long sequence with shared kv heads, ragged
        dict(name='window_train_t4001', kind='window_train', B=1, H=12, Hkv=3, L=4001, window=1000, sinks=1),
        # interactive decoding with a window: one sequence, where latency counts
        dict(name='window_decode_b1', kind='window_decode', dtype='bf16', B=1, H=12, Hkv=3, D=64, L=1, S=4097,
             window=1024, sinks=4),
        # batched decoding with a window over long contexts
        dict(name='window_decode_b64', kind='window_decode', dtype='bf16', B=64, H=12, Hkv=3, D=64, L=1, S=4097,
             window=1024, sinks=4),
        # the rows of one decoding step of a batch
        dict(name='kv4_write_b64_n1', kind='kv4_write', dtype='bf16', B=64, Hkv=3, D=64, cap=4352, start=4096, n=1),
        # the rows of four prompts behind earlier ones
        dict(name='kv4_write_b4_n2048', kind='kv4_write', dtype='bf16', B=4, Hkv=3, D=64, cap=4096, start=1021, n=2048),
        # one short sequence: latency
        dict(name='kv4_decode_b1_s300', kind='kv4_decode', dtype='bf16', B=1, H=12, Hkv=3, D=64, L=1, S=300, cap=512,
             window=0, sinks=0),
        # batched decoding over long contexts: the cache streams through memory
        dict(name='kv4_decode_b64_s4097', kind='kv4_decode', dtype='bf16', B=64, H=12, Hkv=3, D=64, L=1, S=4097,
             cap=4352, window=0, sinks=0),
        # two new tokens of half-precision sequences over longer contexts, with a window
        dict(name='kv4_decode_fp16_s8190', kind='kv4_decode', dtype='fp16', B=32, H=12, Hkv=3, D=64, L=2, S=8190,
             cap=8192, window=4000, sinks=4),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(['window_prefill', 'window_prefill', 'window_train', 'window_decode', 'kv4_write', 'kv4_decode',
                       'kv4_decode'])
    H, Hkv = rng.choice([(12, 3), (12, 12), (8, 2)])
    sinks = rng.choice([0, 1, 4, 16])
    dtype, D = rng.choice(['bf16', 'bf16', 'bf16', 'fp16', 'fp32']), rng.choice([64, 64, 64, 32, 128])
    if kind == 'window_prefill':
        B = rng.choice([1, 1, 2])
        S = _log_int(rng, 33, 4096 if dtype == 'bf16' and D == 64 else 1024)
        return dict(kind=kind, dtype=dtype, B=B, H=H, Hkv=Hkv, D=D, L=S if rng.random() < 0.6 else rng.randint(17, S),
                    S=S, window=_log_int(rng, 16, S), sinks=sinks)
    if kind == 'window_train':
        L = _log_int(rng, 33, 2048)
        return dict(kind=kind, B=rng.choice([1, 2]), H=H, Hkv=Hkv, L=L, window=_log_int(rng, 16, L), sinks=sinks)
    if kind == 'window_decode':
        S = _log_int(rng, 65, 8192)
        return dict(kind=kind, dtype=dtype, B=_log_int(rng, 1, 64 * 3 // Hkv), H=H, Hkv=Hkv, D=D,
                    L=rng.choice([1, 1, 1, 2]), S=S, window=_log_int(rng, 16, min(S, 2048)), sinks=sinks)
    if kind == 'kv4_write':
        B = _log_int(rng, 1, 64)
        n = _log_int(rng, 1, max(1, 8192 // B))
        start = rng.randint(0, 1024)
        return dict(kind=kind, dtype=dtype, B=B, Hkv=Hkv, D=D, cap=start + n + rng.randint(0, 64), start=start, n=n)
    S = _log_int(rng, 65, 8192)
    return dict(kind=kind, dtype=dtype, B=_log_int(rng, 1, 32 * 3 // Hkv), H=H, Hkv=Hkv, D=D, L=rng.choice([1, 1, 1, 2, 3]),
                S=S, cap=S + rng.randint(0, 256), window=0 if rng.random() < 0.5 else _log_int(rng, 16, S), sinks=sinks)


# ------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _attention_inputs(case, seed):
    '''What a Chord layer hands the op: RMS-normalised q and k, positive alpha, small beta
    and mu, ssmax near 1, log_n = ln(position + 1); an output gradient.  q and the gradient
    lie as [B, L, H, D], as a layer has them.'''
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, H, Hkv, L = case['B'], case['H'], case['Hkv'], case['L']
    S, D = case.get('S', L), case.get('D', 64)
    dt = DTYPES[case.get('dtype', 'bf16')]

    def rms(t):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + NORM_EPS)
    q = rms(_randn(g, B, L, H, D)).to(dt).transpose(1, 2)
    k = rms(_randn(g, B, Hkv, S, D)).to(dt)
    v = (0.5 * _randn(g, B, Hkv, S, D)).to(dt)
    par = [torch.exp(0.3 * _randn(g, H)), 0.2 * _randn(g, H), 2 * torch.sinh(0.1 * _randn(g, H)),
           1 + 0.1 * _randn(g, H)]
    log_n = torch.log(torch.arange(S - L + 1, S + 1, dtype=torch.float32, device=DEV))[None].expand(B, L).contiguous()
    do = _randn(g, B, L, H, D).to(dt).transpose(1, 2)
    return q, k, v, par, log_n, do


def _cache_rows(g, B, Hkv, cap, D):
    '''The tensors of a 4-bit cache that a program has filled: codes spread over their
    range, and scale and base of rows near those that the op meets.'''
    codes = torch.randint(0, 256, (B, Hkv, cap, D // 2), generator=g, device=DEV, dtype=torch.uint8)
    G = D // min(GROUP, D)
    scale = 0.25 * (0.5 + torch.rand(B, Hkv, cap, G, generator=g, device=DEV))
    base = -7.5 * scale + 0.2 * _randn(g, B, Hkv, cap, G)
    return codes, torch.stack([scale, base], -1).to(torch.bfloat16)


def prepare(case, seed):
    kind = case['kind']
    st = dict(case)
    if kind.startswith('window'):
        q, k, v, par, log_n, do = _attention_inputs(case, seed)
        if kind == 'window_train':  # (mu is frozen in the layer)
            for t in (q, k, v, par[0], par[1], par[3]):
                t.requires_grad_()
        st.update(q=q, k=k, v=v, par=par, log_n=log_n, do=do)
        return st
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    B, Hkv, D, cap = case['B'], case['Hkv'], case['D'], case['cap']
    st['cache'] = (*_cache_rows(g, B, Hkv, cap, D), *_cache_rows(g, B, Hkv, cap, D))
    if kind == 'kv4_write':
        dt, n = DTYPES[case['dtype']], case['n']
        k = _randn(g, B, n, Hkv, D)
        k = k * torch.rsqrt(k.pow(2).mean(-1, keepdim=True) + NORM_EPS)
        v = 0.5 * _randn(g, B, n, Hkv, D) + 0.1 * _randn(g, Hkv, D)
        st.update(k=k.to(dt).transpose(1, 2), v=v.to(dt).transpose(1, 2))
    else:
        q, _, _, par, log_n, _ = _attention_inputs(case, seed)
        st.update(q=q, par=par, log_n=log_n)
    return st


# ------------------------------------------------------------------ the operators in their plain form
def _attend(q, k, v, par, log_n, window, sinks):
    '''softmax((s q.k + bias) ssmax log_n) v over the visible keys; every tensor fp32, window 0: all.'''
    B, H, L, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    alpha, beta, mu, ssmax = (t.view(H, 1, 1) for t in par)
    kf, vf = (t[:, :, None].expand(B, Hkv, H // Hkv, S, D).reshape(B, H, S, D) for t in (k, v))
    i = torch.arange(S - L, S, device=q.device)[:, None]
    j = torch.arange(S, device=q.device)[None]
    bias = -alpha * (((j - i).float() - mu).abs() + GGD_EPS) ** beta
    z = (torch.matmul(q, kf.transpose(-1, -2).contiguous()) * D ** -0.5 + bias) * (ssmax * log_n[:, None, :, None])
    seen = j <= i
    if window:
        seen = seen & ((j > i - window) | (j < sinks))
    z = z.masked_fill(~seen, float('-inf'))
    e = torch.exp(z - z.amax(-1, keepdim=True))
    return torch.matmul(e / e.sum(-1, keepdim=True), vf)


def _values(codes, params):
    '''The fp32 values of 4-bit rows.'''
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    scale, base = (params[..., m].float().repeat_interleave(c.shape[-1] // params.shape[-2], -1) for m in (0, 1))
    return c * scale + base


def _quantise(x):
    '''(codes, params) of rows x.'''
    grp = min(GROUP, x.shape[-1])
    x = x.float().unflatten(-1, (x.shape[-1] // grp, grp))
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    fifteenth = torch.tensor(1 / 15, dtype=torch.float32, device=x.device)
    scale, base = ((hi - lo) * fifteenth).to(torch.bfloat16), lo.to(torch.bfloat16)
    code = torch.round((x - base.float()) / scale.float()).clamp(0, 15)
    code = torch.where(scale == 0, 0, code).to(torch.uint8).flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), torch.cat([scale, base], -1)


def run(state):
    kind = state['kind']
    if own:
        return _run_own(state)
    if kind == 'window_train':
        q, k, v, par, log_n = (state[n] for n in ('q', 'k', 'v', 'par', 'log_n'))
        o = _attend(q.float(), k.float(), v.float(), par, log_n, state['window'], state['sinks']).to(q.dtype)
        return [o.detach(), *torch.autograd.grad(o, (q, k, v, par[0], par[1], par[3]), state['do'])]
    with torch.no_grad():
        if kind.startswith('window'):
            q, k, v = state['q'], state['k'], state['v']
            return _attend(q.float(), k.float(), v.float(), state['par'], state['log_n'], state['window'],
                           state['sinks']).to(q.dtype)
        kc, kp, vc, vp = state['cache']
        if kind == 'kv4_write':
            rows = slice(state['start'], state['start'] + state['n'])
            kc[:, :, rows], kp[:, :, rows] = _quantise(state['k'])
            vc[:, :, rows], vp[:, :, rows] = _quantise(state['v'])
            dt = state['k'].dtype
            return [_values(kc[:, :, rows], kp[:, :, rows]).to(dt), _values(vc[:, :, rows], vp[:, :, rows]).to(dt)]
        S, q = state['S'], state['q']
        k, v = _values(kc[:, :, :S], kp[:, :, :S]), _values(vc[:, :, :S], vp[:, :, :S])
        return _attend(q.float(), k, v, state['par'], state['log_n'], state['window'], state['sinks']).to(q.dtype)


# ------------------------------------------------------------------ the framework's own
def _run_own(state):
    if os.path.join(os.getcwd(), 'codon-motif_amd') not in sys.path:
        sys.path.insert(0, os.path.join(os.getcwd(), 'codon-motif_amd'))
    from motif.ops import KV4Slab, apply_chord_attention, chord_attention_kv4, kv4_append, kv4_read
    kind = state['kind']
    if kind == 'window_train':
        q, k, v, par, log_n = (state[n] for n in ('q', 'k', 'v', 'par', 'log_n'))
        o = apply_chord_attention(q, k, v, *par, log_n, window=state['window'], sinks=state['sinks'])
        return [o.detach(), *torch.autograd.grad(o, (q, k, v, par[0], par[1], par[3]), state['do'])]
    with torch.no_grad():
        if kind.startswith('window'):
            return apply_chord_attention(state['q'], state['k'], state['v'], *state['par'], state['log_n'],
                                         window=state['window'], sinks=state['sinks'])
        slab = KV4Slab(*state['cache'])
        if kind == 'kv4_write':
            kv4_append(slab, state['k'], state['v'], state['start'])
            return list(kv4_read(slab, state['start'], state['n'], state['k'].dtype))
        return chord_attention_kv4(state['q'], slab, *state['par'], state['log_n'], state['S'],
                                   window=state['window'] or None, sinks=state['sinks'] if state['window'] else 0)


# ------------------------------------------------------------------ what a pass cannot do without
def _seen(L, S, window, sinks):
    '''(visible (query, key) pairs, keys that any query sees) of L queries that end at position S.'''
    if not window:
        return L * (S - L) + L * (L + 1) // 2, S
    pairs = 0
    for p in range(S - L, S):
        lo = max(0, p - window + 1)
        pairs += p + 1 - lo + min(sinks, lo)
    lo = max(0, S - L - window + 1)
    return pairs, S - lo + min(sinks, lo)


def work(case):
    kind, B, Hkv = case['kind'], case['B'], case['Hkv']
    D, e = case.get('D', 64), DTYPES[case.get('dtype', 'bf16')].itemsize
    row4 = D // 2 + 4 * (D // min(GROUP, D))
    if kind == 'kv4_write':
        rows = 2 * B * Hkv * case['n']
        return dict(bytes=rows * (2 * D * e + 2 * row4), flops=8 * D * rows)
    H, L = case['H'], case['L']
    S = case.get('S', L)
    pairs, keys = _seen(L, S, case['window'], case['sinks'])
    nq, nkv = B * H * L * D, B * Hkv * keys * D
    if kind == 'window_train':  # forward, then inputs, output and dO and a gradient per input
        return dict(bytes=e * (2 * nq + 2 * nkv + 4 * nq + 4 * nkv), flops=14 * D * B * H * pairs)
    kv = 2 * B * Hkv * keys * row4 if kind == 'kv4_decode' else 2 * e * nkv
    return dict(bytes=2 * e * nq + kv, flops=4 * D * B * H * pairs)


# ------------------------------------------------------------------ the same in 64 bits
def _head64(q, k, v, p, log_n, window, sinks, do=None):
    '''One head of one batch row from the definition, and with `do` its gradients
    (dq, dk, dv, dalpha, dbeta, dssmax).'''
    L, D = q.shape
    S = k.shape[0]
    q, k, v, log_n = q.double(), k.double(), v.double(), log_n.double()
    al, be, mu, ss = (float(t) for t in p)
    pos = torch.arange(S - L, S, device=q.device, dtype=torch.float64)
    dist = torch.arange(S, device=q.device, dtype=torch.float64) - pos[:, None]
    x = (dist - mu).abs() + GGD_EPS
    xb = torch.exp(be * torch.log(x))
    r = q @ k.T / math.sqrt(D) - al * xb
    c = (ss * log_n)[:, None]
    keep = dist <= 0
    if window:
        first = torch.arange(S, device=q.device) < sinks
        keep &= (dist > -window) | first
    P = torch.softmax(torch.where(keep, c * r, torch.tensor(-math.inf, dtype=torch.float64, device=q.device)), -1)
    o = P @ v
    if do is None:
        return o
    do = do.double()
    dz = P * (do @ v.T - (do * o).sum(-1, keepdim=True))
    cdz = c * dz
    return [o, cdz @ k / math.sqrt(D), cdz.T @ q / math.sqrt(D), P.T @ do, -(cdz * xb).sum(),
            -(cdz * al * xb * torch.log(x)).sum(), (log_n[:, None] * dz * r).sum()]


def _heads64(q, k, v, par, log_n, window, sinks, do=None):
    B, H, L, D = q.shape
    Hkv = k.shape[1]
    got = [[_head64(q[b, h], k[b, h * Hkv // H], v[b, h * Hkv // H], [t[h] for t in par], log_n[b], window, sinks,
                    None if do is None else do[b, h]) for h in range(H)] for b in range(B)]
    if do is None:
        return torch.stack([torch.stack(row) for row in got])
    o, dq, dk, dv, da, db, ds = (torch.stack([torch.stack([x[m] for x in row]) for row in got]) for m in range(7))
    dk, dv = (t.view(B, Hkv, H // Hkv, -1, D).sum(2) for t in (dk, dv))
    return [o, dq, dk, dv, da.sum(0), db.sum(0), ds.sum(0)]


def _values64(codes, params):
    out = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    out[..., 0::2], out[..., 1::2] = codes % 16, codes // 16
    grp = out.unflatten(-1, (params.shape[-2], -1))
    return (grp * params[..., :1].double() + params[..., 1:].double()).flatten(-2)


def _rows64(x):
    '''The values that the codes of rows x stand for: scale and base as they are held (bf16), the codes chosen in 64 bits.'''
    g = x.double().unflatten(-1, (-1, min(GROUP, x.shape[-1])))
    lo = g.amin(-1, keepdim=True)
    scale = ((g.amax(-1, keepdim=True) - lo) / 15).to(torch.bfloat16).double()
    lo = lo.to(torch.bfloat16).double()
    code = torch.where(scale > 0, (g - lo) / scale, 0.0).round().clamp(0, 15)
    return (code * scale + lo).flatten(-2)


@torch.no_grad()
def exact(case, seed):
    kind = case['kind']
    if kind.startswith('window'):
        q, k, v, par, log_n, do = _attention_inputs(case, seed)
        return _heads64(q, k, v, par, log_n, case['window'], case['sinks'], do if kind == 'window_train' else None)
    st = prepare(case, seed)
    if kind == 'kv4_write':
        return [_rows64(st['k']), _rows64(st['v'])]
    kc, kp, vc, vp = (t[:, :, :case['S']] for t in st['cache'])
    return _heads64(st['q'], _values64(kc, kp), _values64(vc, vp), st['par'], st['log_n'], case['window'], case['sinks'])
