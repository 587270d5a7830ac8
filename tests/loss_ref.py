'''64-bit forms of linear_cross_entropy, the row norms and dropout, and how far kernels that
round as theirs do may be from them (elementwise bounds).'''
import numpy as np
import torch

U = 2.0 ** -24  # half a step of fp32


def half(dt):
    '''The most that rounding to dt changes a value by, relative to it.'''
    return torch.finfo(dt).eps / 2


def ce64(x, w, labels, dloss=None, reduction='mean', ignore=-100):
    '''(losses as linear_cross_entropy returns them, dx, dw, bounds of each) in float64.

    Bounds: z is a sum of d products in fp32: off by at most (d + 2) U sum |x w|.  The
    log-sum-exp moves by no more than its z, and by the fp32 sum of positive terms, at
    most 64 + V / 64 of them after each other, each an exponential good to 4 U beside an
    argument rounded at the size of z.  P moves by softmax times both, and is rounded to
    x's type for the products; those add up to V (or N) terms in fp32; dx and dw are rounded once.'''
    dt = x.dtype
    N, d = x.shape
    V = w.shape[0]
    x64, w64 = x.detach().double(), w.detach().double()
    live = labels != ignore
    xs, ts = x64[live], labels[live]
    n = len(ts)
    z = xs @ w64.T
    lse = torch.logsumexp(z, -1)
    rows = lse - z.gather(1, ts[:, None])[:, 0]
    size = (xs.abs() @ w64.abs().T).amax(-1) if n else lse
    delta = 2 * (d + 4) * U * size + (96 + V / 64) * U + 8 * U * z.abs().amax(-1) if n else lse
    loss = torch.zeros(N, dtype=torch.float64, device=x.device)
    tol = torch.zeros_like(loss)
    loss[live], tol[live] = rows, 2 * delta + 4 * U * (lse.abs() + rows.abs())
    if reduction != 'none':
        k = n if reduction == 'mean' else 1
        loss, tol = loss.sum() / k, tol.sum() / k + 2 * U * (loss.sum() / k).abs()
    if dloss is None:
        return loss, tol
    s = dloss.double().expand(N)[live] if reduction == 'none' else dloss.double().expand(n)
    s = s / n if reduction == 'mean' else s
    soft = torch.exp(z - lse[:, None])
    P = soft.clone()
    P[torch.arange(n, device=x.device), ts] -= 1
    P, soft = P * s[:, None], soft * s.abs()[:, None]
    # |error of P|: its rounding, two fp32 roundings of it, and softmax's
    off = (half(dt) + 4 * U) * P.abs() + soft * (2 * delta[:, None] + 8 * U)
    dx, tx = torch.zeros_like(x64), torch.zeros_like(x64)
    dx[live], tx[live] = P @ w64, (off + V * U * P.abs()) @ w64.abs()
    dw, tw = P.T @ xs, (off + (n + 4) * U * P.abs()).T @ xs.abs()
    tiny = torch.finfo(dt).tiny
    return loss, tol, dx, tx + half(dt) * dx.abs() + tiny, dw, tw + half(dt) * dw.abs() + tiny


def norm64(x, w, b, dy, eps, layer):
    '''[(y, bound), (dx, bound), (dw, bound), (db, bound)] in float64 of rows x [N, D].

    Bounds: a sum of D terms in fp32 is off by D U times the sum of their sizes: that moves
    the mean by D U mean|x|, r by (D + 8) U relative (and by the mean's error, of second order
    around the mean); h = (x - m) r by both; y, dx, dw, db follow term by term and are rounded once.'''
    dt = x.dtype
    N, D = x.shape
    x, dy = x.detach().double(), dy.double()
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    bb = torch.zeros_like(w) if b is None else b.detach().double()
    m = x.mean(-1, keepdim=True) if layer else torch.zeros_like(x[:, :1])
    c = x - m
    r = 1 / torch.sqrt(c.square().mean(-1, keepdim=True) + eps)
    h = c * r
    g = dy * w
    gh, g0 = (g * h).mean(-1, keepdim=True), g.mean(-1, keepdim=True) * layer
    e_m = (D + 2) * U * x.abs().mean(-1, keepdim=True) * layer
    e_h = (D + 12) * U * h.abs() + (e_m + 2 * U * (x.abs() + m.abs()) * layer) * r
    y = h * w + bb
    e_y = e_h * w.abs() + 4 * U * (y.abs() + (h * w).abs())
    e_gh = (D + 4) * U * (g * h).abs().mean(-1, keepdim=True) + (g.abs() * e_h).mean(-1, keepdim=True)
    e_g0 = (D + 4) * U * g.abs().mean(-1, keepdim=True) * layer
    inner = g - h * gh - g0
    e_dx = r * (e_gh * h.abs() + gh.abs() * e_h + e_g0 + (D + 20) * U * (g.abs() + (h * gh).abs() + g0.abs()))
    dx = r * inner
    dw, e_dw = (dy * h).sum(0), (dy.abs() * e_h).sum(0) + (N + 4) * U * (dy * h).abs().sum(0)
    db, e_db = dy.sum(0), (N + 4) * U * dy.abs().sum(0)
    tiny = torch.finfo(dt).tiny
    out = [(v, e + half(dt) * v.abs() + tiny) for v, e in ((y, e_y), (dx, e_dx), (dw, e_dw), (db, e_db))]
    return out


def kept(n, seed, p, first=0):
    '''Which of the elements first .. first + n - 1 are kept (first a multiple of 4), from the definition.'''
    u, low, sh = np.uint64, np.uint64(0xffffffff), np.uint64(32)
    i = np.arange(first // 4, first // 4 + -(-n // 4), dtype=np.uint64)
    c = [i & low, i >> sh, np.zeros_like(i), np.zeros_like(i)]
    key = [seed & 0xffffffff, (seed >> 32) & 0xffffffff]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> sh) ^ c[1] ^ u(key[0]), b & low, (a >> sh) ^ c[3] ^ u(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) & 0xffffffff, (key[1] + 0xBB67AE85) & 0xffffffff]
    return torch.from_numpy(np.stack(c, 1).reshape(-1)[:n] >= u(int(round(p * 2 ** 32))))


def check(got, want, tol, what):
    '''Every element of got within tol of want.'''
    got, want = got.detach().double(), want.to(got.device)
    assert got.shape == want.shape, f'{what}: {tuple(got.shape)} for {tuple(want.shape)}'
    bad = ~((got - want).abs() <= tol)
    if bool(bad.any()):
        at = bad.nonzero()[0].tolist()
        i = tuple(at)
        t = tol[i] if isinstance(tol, torch.Tensor) and tol.dim() else tol
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} outside, first at {at}: '
                             f'{got[i].item():.9g} for {want[i].item():.9g} (bound {float(t):.3g})')
