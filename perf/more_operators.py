'''The operators around a training step's mixers: the loss straight from the hidden states, the
row norms and dropout with their gradients: the calls that a program makes of them, for timing
and comparison.

  ce_train   linear_cross_entropy, mean over the rows, forward and backward
  ce_score   linear_cross_entropy, one loss per row, forward only
  rms        rms_norm_rows forward and backward (input and weight)
  layer      layer_norm_rows forward and backward (input, weight and bias)
  dropout    dropout_add forward and backward (with or without a residual)

linear_cross_entropy: row i of x [N, d] with label t_i has the loss
  log sum_v exp(x_i . w_v) - x_i . w_{t_i}  over the rows w_v of weight [V, d];
rows whose label is -100 count nothing and get no gradient.

rms_norm_rows: y = x / sqrt(mean(x^2) + eps) * w; layer_norm_rows: y = (x - mean) / sqrt(var + eps) * w + b.

dropout_add: y = residual + x * keep / (1 - p).  Element e of x (row-major) is kept when word
e mod 4 of Philox4x32-10 (Salmon et al., SC 2011) at counter (e div 4 as two 32-bit words, 0, 0)
under the 64-bit key `seed` is at least round(p 2^32).

Sizes: 768 features, heads of 64, a vocabulary of 32000 or 40960, 4096 tokens and batches of four
are the 172M model's and the benchmark's; the rest are generic.
'''
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = 'cuda'
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
IGNORE = -100
EPS = {'rms': 1e-6, 'layer': 1e-5}


def listed():
    return [
        # the loss of a training step over one 4096-token sequence
        dict(name='ce_train_t4096', kind='ce_train', dtype='bf16', N=4096, d=768, V=32000, ignored=0.0),
        # four such sequences, the default vocabulary, some padding: the largest pass
        dict(name='ce_train_b4_t4096', kind='ce_train', dtype='bf16', N=16384, d=768, V=40960, ignored=0.05),
        # fine-tuning on answers: most rows are prompt and carry no label, ragged
        dict(name='ce_train_answers', kind='ce_train', dtype='bf16', N=2111, d=768, V=32000, ignored=0.7),
        # the accuracy mode at a small model, odd sizes
        dict(name='ce_train_fp32', kind='ce_train', dtype='fp32', N=301, d=256, V=5003, ignored=0.1),
        # scoring one text: the log probability of each token
        dict(name='ce_score_t517', kind='ce_score', dtype='bf16', N=517, d=768, V=32000, ignored=0.0),
        # a decoder's input norm over four sequences
        dict(name='rms_t16384', kind='rms', dtype='bf16', N=16384, D=768),
        # the query norm of a Chord layer: a row for each of 12 heads
        dict(name='rms_heads', kind='rms', dtype='bf16', N=49152, D=64),
        # one short sequence: latency
        dict(name='rms_t64', kind='rms', dtype='bf16', N=64, D=768),
        # a layer norm in the accuracy mode, odd sizes
        dict(name='layer_fp32_odd', kind='layer', dtype='fp32', N=1001, D=771),
        # wide rows, many of them
        dict(name='layer_wide', kind='layer', dtype='bf16', N=8192, D=2048),
        # a residual branch of four sequences
        dict(name='dropout_t16384', kind='dropout', dtype='bf16', N=16384, D=768, p=0.1, residual=True),
        # a small fp32 tensor of odd size
        dict(name='dropout_fp32_odd', kind='dropout', dtype='fp32', N=999, D=257, p=0.5, residual=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(['ce_train', 'ce_train', 'ce_score', 'rms', 'layer', 'dropout'])
    if kind.startswith('ce'):
        dtype = rng.choice(['bf16', 'bf16', 'bf16', 'fp32'])
        d = rng.choice([64, 100, 200, 256, 768, 768, 1024])
        N = _log_int(rng, 1, 8192 if dtype == 'bf16' else 512)
        V = _log_int(rng, 257, 40960 if dtype == 'bf16' else 8192)
        return dict(kind=kind, dtype=dtype, N=N, d=d, V=V, ignored=rng.choice([0.0, 0.0, 0.1, 0.6]))
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    D = rng.choice([64, 128, 768, 768, 1024, _log_int(rng, 16, 8192)])
    N = _log_int(rng, 1, (1 << 24) // D)
    if kind == 'dropout':
        return dict(kind=kind, dtype=dtype, N=N, D=D, p=rng.choice([0.05, 0.1, 0.3, 0.5]), residual=rng.random() < 0.5)
    return dict(kind=kind, dtype=dtype, N=N, D=D)


# ------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, dt, st = case['kind'], DTYPES[case['dtype']], dict(case)
    if kind.startswith('ce'):
        N, d, V = case['N'], case['d'], case['V']
        w = (0.05 * _randn(g, V, d)).to(dt)
        labels = torch.randint(0, V, (N,), generator=g, device=DEV)
        # normalised hidden states that favour the label, some rows strongly
        t = w[labels].float()
        boost = 12 * torch.rand(N, 1, generator=g, device=DEV)
        x = (_randn(g, N, d) + boost * t / t.pow(2).sum(-1, keepdim=True)).to(dt)
        drop = torch.rand(N, generator=g, device=DEV) < case['ignored']
        drop[:1] = False  # (a step has at least one label)
        labels = torch.where(drop, IGNORE, labels)
        if kind == 'ce_train':
            x.requires_grad_()
            w.requires_grad_()
        st.update(x=x, w=w, labels=labels)
        return st
    N, D = case['N'], case['D']
    st['x'] = (1.5 * _randn(g, N, D) + 0.1).to(dt).requires_grad_()
    st['dy'] = _randn(g, N, D).to(dt)
    if kind == 'dropout':
        st['res'] = _randn(g, N, D).to(dt).requires_grad_() if case['residual'] else None
        st['seed'] = torch.randint(0, 2 ** 62, (1,), generator=g, device=DEV)
        return st
    st['w'] = (1 + 0.1 * _randn(g, D)).to(dt).requires_grad_()
    if kind == 'layer':
        st['b'] = (0.1 * _randn(g, D)).to(dt).requires_grad_()
    return st


# ------------------------------------------------------------------ the operators in their plain form
def _row_losses(x, w, labels):
    '''(loss of each row, 0 where it has no label; which rows have one)'''
    logits = x.float() @ w.float().t()
    top = logits.amax(-1, keepdim=True)
    lse = torch.log(torch.exp(logits - top).sum(-1)) + top[:, 0]
    valid = labels != IGNORE
    at = logits.gather(1, torch.where(valid, labels, 0)[:, None])[:, 0]
    return torch.where(valid, lse - at, 0.0), valid


def _philox(counter, key_lo, key_hi):
    '''The four words (int64 tensors of 32-bit values) of Philox4x32-10 at 64-bit counters.'''
    low = 0xffffffff
    c = [counter & low, (counter >> 32) & low, torch.zeros_like(counter), torch.zeros_like(counter)]
    k0, k1 = key_lo, key_hi
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # (the wrapped products hold all 64 bits)
        c = [((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c


def _kept(n, seed, p, device):
    '''Which of n elements are kept.'''
    counter = torch.arange((n + 3) // 4, device=device)
    words = _philox(counter, seed & 0xffffffff, (seed >> 32) & 0xffffffff)
    return torch.stack(words, -1).flatten()[:n] >= int(round(p * 2 ** 32))


def run(state):
    kind = state['kind']
    if own:
        return _run_own(state)
    if kind == 'ce_score':
        with torch.no_grad():
            return _row_losses(state['x'], state['w'], state['labels'])[0]
    if kind == 'ce_train':
        rows, valid = _row_losses(state['x'], state['w'], state['labels'])
        loss = rows.sum() / valid.sum()
        return [loss.detach(), *torch.autograd.grad(loss, (state['x'], state['w']))]
    x, dy = state['x'], state['dy']
    xf = x.float()
    if kind == 'dropout':
        keep = _kept(x.numel(), state['seed'], state['p'], x.device).view(x.shape)
        y = torch.where(keep, xf * (1 / (1 - state['p'])), 0.0)
        if state['res'] is None:
            y = y.to(x.dtype)
            return [y.detach(), *torch.autograd.grad(y, (x,), dy)]
        y = (state['res'].float() + y).to(x.dtype)
        return [y.detach(), *torch.autograd.grad(y, (x, state['res']), dy)]
    if kind == 'rms':
        y = (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + EPS[kind]) * state['w'].float()).to(x.dtype)
        return [y.detach(), *torch.autograd.grad(y, (x, state['w']), dy)]
    z = xf - xf.mean(-1, keepdim=True)
    z = z * torch.rsqrt(z.pow(2).mean(-1, keepdim=True) + EPS[kind])
    y = (z * state['w'].float() + state['b'].float()).to(x.dtype)
    return [y.detach(), *torch.autograd.grad(y, (x, state['w'], state['b']), dy)]


# ------------------------------------------------------------------ the framework's own
def _run_own(state):
    if os.path.join(os.getcwd(), 'codon-motif_amd') not in sys.path:
        sys.path.insert(0, os.path.join(os.getcwd(), 'codon-motif_amd'))
    from motif.ops import dropout_add, layer_norm_rows, linear_cross_entropy, rms_norm_rows
    kind, x = state['kind'], state['x']
    if kind == 'ce_score':
        with torch.no_grad():
            return linear_cross_entropy(x, state['w'], state['labels'], ignore_index=IGNORE, reduction='none')
    if kind == 'ce_train':
        loss = linear_cross_entropy(x, state['w'], state['labels'], ignore_index=IGNORE)
        return [loss.detach(), *torch.autograd.grad(loss, (x, state['w']))]
    if kind == 'dropout':
        y = dropout_add(x, state['p'], state['seed'], residual=state['res'])
        leaves = (x,) if state['res'] is None else (x, state['res'])
    elif kind == 'rms':
        y = rms_norm_rows(x, state['w'], EPS[kind])
        leaves = (x, state['w'])
    else:
        y = layer_norm_rows(x, state['w'], state['b'], EPS[kind])
        leaves = (x, state['w'], state['b'])
    return [y.detach(), *torch.autograd.grad(y, leaves, state['dy'])]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    kind, e, N = case['kind'], DTYPES[case['dtype']].itemsize, case['N']
    if kind.startswith('ce'):
        d, V = case['d'], case['V']
        rows = N * (1 - case['ignored'])  # a row without a label is not multiplied
        if kind == 'ce_score':
            return dict(bytes=e * (N * d + V * d) + 12 * N, flops=2 * rows * d * V)
        return dict(bytes=2 * e * (N * d + V * d) + 8 * N, flops=6 * rows * d * V)
    n = N * case['D']
    if kind == 'dropout':  # x (and the residual) in, y out; dy in, dx out (the residual's gradient is dy)
        return dict(bytes=e * n * (5 if case['residual'] else 4), flops=4 * n)
    vec = 4 if kind == 'layer' else 2
    return dict(bytes=e * (5 * n + (vec + 1) * case['D']), flops=14 * n)  # x in, y out; x and dy in, dx out


# ------------------------------------------------------------------ the same in 64 bits
def _kept_np(n, key, p):
    '''Which of n elements are kept, in numpy's unsigned 64-bit words.'''
    u = np.uint64
    low, sh = u(0xffffffff), u(32)
    idx = np.arange(-(-n // 4), dtype=np.uint64)
    x0, x1 = idx & low, idx >> sh
    x2 = x3 = np.zeros_like(idx)
    ka, kb = key & 0xffffffff, key >> 32
    for r in range(10):
        p0, p1 = u(0xD2511F53) * x0, u(0xCD9E8D57) * x2
        ra, rb = u((ka + r * 0x9E3779B9) & 0xffffffff), u((kb + r * 0xBB67AE85) & 0xffffffff)
        x0, x1, x2, x3 = (p1 >> sh) ^ x1 ^ ra, p1 & low, (p0 >> sh) ^ x3 ^ rb, p0 & low
    words = np.empty((len(idx), 4), dtype=np.uint64)
    for m, wd in enumerate((x0, x1, x2, x3)):
        words[:, m] = wd
    return words.reshape(-1)[:n] >= u(int(round(p * 2 ** 32)))


@torch.no_grad()
def _ce64(x, w, labels, train):
    x, w = x.detach().double(), w.detach().double()
    rows = torch.zeros(len(x), dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    live = (labels != IGNORE).nonzero()[:, 0]
    for part in live.split(2048):
        z = x[part] @ w.T
        lse = torch.logsumexp(z, -1)
        rows[part] = lse - z[torch.arange(len(part), device=x.device), labels[part]]
        if train:
            z = torch.exp(z - lse[:, None])
            z[torch.arange(len(part), device=x.device), labels[part]] -= 1
            z /= len(live)
            dx[part] = z @ w
            dw += z.T @ x[part]
    return [rows.sum() / len(live), dx, dw] if train else rows


@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    kind = case['kind']
    if kind.startswith('ce'):
        return _ce64(st['x'], st['w'], st['labels'], kind == 'ce_train')
    x, dy = st['x'].double(), st['dy'].double()
    if kind == 'dropout':
        keep = torch.from_numpy(_kept_np(x.numel(), int(st['seed']), case['p'])).to(x.device).view(x.shape)
        f = keep.double() / (1 - case['p'])
        return [x * f, dy * f] if st['res'] is None else [st['res'].double() + x * f, dy * f, dy]
    w = st['w'].double()
    c = x - x.mean(-1, keepdim=True) if kind == 'layer' else x
    r = 1 / torch.sqrt(c.square().mean(-1, keepdim=True) + EPS[kind])
    h, g = c * r, dy * w
    dx = g - h * (g * h).mean(-1, keepdim=True)
    if kind == 'rms':
        return [h * w, r * dx, (dy * h).sum(0)]
    return [h * w + st['b'].double(), r * (dx - g.mean(-1, keepdim=True)), (dy * h).sum(0), dy.sum(0)]
