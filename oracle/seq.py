"""The causal sequence operators in 64 bits on the CPU, from their formulas, one frame at a time (test infrastructure only).

Each function returns a dict of results; with ``mag=True`` every term enters by its absolute value, so that the result bounds the sum of
the absolute values of the terms that the true result adds up - what a rounding error in 32 bits is relative to.
Philox-4x32-10 is the published generator (J. Salmon et al., SC 2011), pinned by that paper's known answers in tests/test_seq.py.
"""
import math

import torch


def _silu(v, mag):
    s = torch.sigmoid(v)
    g, d = v * s, s * (1 + v * (1 - s))
    return (g.abs(), s * (1 + v.abs() * (1 - s))) if mag else (g, d)


def conv(x, w, b=None, silu=True, lengths=None, state=None, dy=None, mag=False):
    x, w = x.double(), w.double()
    T, N, C = x.shape
    K = w.shape[1]
    n = lengths if lengths is not None else torch.full((N,), T)
    on = (torch.arange(T).unsqueeze(1) < n.clamp(0, T)).unsqueeze(2)
    x = torch.where(on, x, torch.zeros_like(x))
    past = torch.zeros(K - 1, N, C, dtype=torch.float64) if state is None else state.double().transpose(0, 1)
    X = torch.cat([past, x])
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.double()
    p = b + sum(X[k:k + T] * w[:, k] for k in range(K))
    pm = b.abs() + sum((X[k:k + T] * w[:, k]).abs() for k in range(K))
    y, slope = _silu(p, False) if silu else (p, torch.ones_like(p))
    zero = torch.zeros_like(p)
    if mag:                                # |d silu| <= 1.1: an error of p passes on by at most that, |d slope| <= 0.5
        y = 1.1 * pm if silu else pm
    out = dict(y=torch.where(on, y, zero))
    at = n.clamp(0, T).long().unsqueeze(0) + torch.arange(K - 1).unsqueeze(1)
    out["state"] = X.gather(0, at.unsqueeze(2).expand(-1, -1, C)).transpose(0, 1).contiguous()
    if dy is not None:
        dy = torch.where(on, dy.double(), zero)
        g = dy * slope
        if mag:
            g, X, w = dy.abs() * (1.1 + 0.5 * pm if silu else 1.0), X.abs(), w.abs()
        after = torch.cat([g, torch.zeros(K - 1, N, C, dtype=torch.float64)])
        out["dx"] = torch.where(on, sum(after[K - 1 - k:K - 1 - k + T] * w[:, k] for k in range(K)), zero)
        out["dw"] = torch.stack([(g * X[k:k + T]).sum((0, 1)) for k in range(K)], 1)
        out["db"] = g.sum((0, 1))
    return out


def scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, lengths=None, state=None, dy=None, mag=False):
    x, dt, A, B, C = (v.double() for v in (x, dt, A, B, C))
    if B.dim() == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    T, N, Ch = x.shape
    S, G = A.shape[1], B.shape[2]
    n = (lengths if lengths is not None else torch.full((N,), T)).clamp(0, T)
    on = (torch.arange(T).unsqueeze(1) < n).unsqueeze(2)
    fix = lambda v: torch.where(on if v.dim() == 3 else on.unsqueeze(3), v, torch.zeros_like(v))
    x, dt, B, C = fix(x), fix(dt), fix(B), fix(C)
    pre = dt + (0 if dt_bias is None else dt_bias.double())
    d = torch.logaddexp(pre, torch.zeros_like(pre)) if softplus else pre
    dslope = torch.sigmoid(pre) if softplus else torch.ones_like(pre)
    Dv = torch.zeros(Ch, dtype=torch.float64) if D is None else D.double()
    gate, gslope = (torch.ones_like(x), torch.zeros_like(x)) if z is None else _silu(fix(z.double()), mag)
    if mag:
        x, B, C, Dv = x.abs(), B.abs(), C.abs(), Dv.abs()
    Bc, Cc = B.repeat_interleave(Ch // G, 2), C.repeat_interleave(Ch // G, 2)
    da = d.abs() if mag else d
    h = torch.zeros(N, Ch, S, dtype=torch.float64) if state is None else state.double().clone()
    h = h.abs() if mag else h
    hs, prev = [], []
    for t in range(T):
        prev.append(h)
        new = torch.exp(d[t].unsqueeze(-1) * A) * h + (da[t] * x[t]).unsqueeze(-1) * Bc[t]
        h = torch.where(on[t].unsqueeze(-1), new, h)
        hs.append(h)
    empty = torch.zeros(0, N, Ch, S, dtype=torch.float64)
    H, P = (torch.stack(v) if T else empty for v in (hs, prev))
    o = (H * Cc).sum(-1) + Dv * x
    out = dict(y=fix(o * gate), state=h)
    if dy is None:
        return out
    dy = fix(dy.double())
    dy = dy.abs() if mag else dy
    go = dy * gate
    out["dz"] = dy * o * gslope
    dx, dd = torch.zeros_like(x), torch.zeros_like(x)
    out["dA"], dBc, dCc = torch.zeros_like(A), torch.zeros_like(Bc), torch.zeros_like(Cc)
    carry = torch.zeros(N, Ch, S, dtype=torch.float64)
    Aa = A.abs() if mag else A
    for t in reversed(range(T)):
        a = torch.exp(d[t].unsqueeze(-1) * A)
        g = carry + go[t].unsqueeze(-1) * Cc[t]
        g = torch.where(on[t].unsqueeze(-1), g, torch.zeros_like(g))
        q = g * a * P[t]
        out["dA"] += (q * da[t].unsqueeze(-1)).sum(0)
        u = (g * Bc[t]).sum(-1)
        dx[t] = u * da[t] + go[t] * Dv
        dd[t] = ((q * Aa).sum(-1) + u * x[t]) * dslope[t]
        dBc[t] = g * (da[t] * x[t]).unsqueeze(-1)
        dCc[t] = go[t].unsqueeze(-1) * H[t]
        carry = g * a
    out["dx"], out["ddt"] = fix(dx), fix(dd)
    out["ddt_bias"] = out["ddt"].sum((0, 1))
    out["dD"] = (go * x).sum((0, 1))
    out["dB"] = fix(dBc.view(T, N, G, Ch // G, S).sum(3))
    out["dC"] = fix(dCc.view(T, N, G, Ch // G, S).sum(3))
    return out


def philox(counter, key):
    """One block: counter (4 words), key (2 words) -> 4 words; Python integers."""
    c, k, m = list(counter), list(key), 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & m, (a >> 32) ^ c[3] ^ k[1], a & m]
        k = [(k[0] + 0x9E3779B9) & m, (k[1] + 0xBB67AE85) & m]
    return c


def keep_mask(n, p, seed, offset=0):
    """Truth values [n]: the elements that dropout keeps."""
    thr, m = int(math.floor(p * 65536 + 0.5)), 0xFFFFFFFF
    bits = []
    for j in range((n + 7) // 8):
        c = (offset + j) % 2 ** 64
        for w in philox((c & m, c >> 32, 0, 0), (seed & m, (seed % 2 ** 64) >> 32)):
            bits += [w & 0xFFFF, w >> 16]
    return torch.tensor(bits[:n]) >= thr


def drop_factor(p):
    thr = int(math.floor(p * 65536 + 0.5))
    return 0.0 if thr >= 65536 else 65536.0 / (65536 - thr)


def dropout(x, p, seed, offset=0):
    keep = keep_mask(x.numel(), p, seed, offset).view(x.shape)
    return torch.where(keep, x.double() * drop_factor(p), torch.zeros_like(x, dtype=torch.float64))


def residual_norm(x, residual=None, weight=None, bias=None, scale=None, eps=1e-5, kind="rms", p=0.0, seed=0, offset=0, kept=None, dy=None, dr=None):
    """Gradients by torch's own differentiation of the definition.  kept: r as it was stored (a rounding of this r), which the norm
    reads and which passes gradients unchanged."""
    leaf = lambda v: None if v is None else v.detach().double().requires_grad_()
    x, residual, weight, bias, scale = (leaf(v) for v in (x, residual, weight, bias, scale))
    b = x
    if p:
        keep = keep_mask(x.numel(), p, seed, offset).view(x.shape)
        b = torch.where(keep, x * drop_factor(p), torch.zeros_like(x))
    r = b if scale is None else b * scale
    r = r if residual is None else residual + r
    kept = r if kept is None else r + (kept.double() - r.detach())
    v = kept - kept.mean(-1, keepdim=True) if kind == "layer" else kept
    y = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
    y = y if weight is None else y * weight
    y = y if bias is None else y + bias
    out = dict(y=y.detach(), r=r.detach())
    if dy is not None or dr is not None:
        names = [(n, t) for n, t in (("dx", x), ("dresidual", residual), ("dweight", weight), ("dbias", bias), ("dscale", scale)) if t is not None]
        given = [(o, g.double()) for o, g in ((y, dy), (r, dr)) if g is not None]
        grads = torch.autograd.grad([o for o, _ in given], [t for _, t in names], [g for _, g in given], allow_unused=True)
        out.update({n: torch.zeros_like(t) if g is None else g for (n, t), g in zip(names, grads)})
    return out


def gated_norm(x, gate, weight=None, eps=1e-5, groups=1, norm_first=False, dy=None):
    leaf = lambda v: None if v is None else v.detach().double().requires_grad_()
    x, gate, weight = leaf(x), leaf(gate), leaf(weight)
    g = gate * torch.sigmoid(gate)
    v = (x if norm_first else x * g).unflatten(-1, (groups, -1))
    y = (v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)).flatten(-2)
    y = y if weight is None else y * weight
    y = y * g if norm_first else y
    out = dict(y=y.detach())
    if dy is not None:
        names = [(n, t) for n, t in (("dx", x), ("dgate", gate), ("dweight", weight)) if t is not None]
        out.update(zip([n for n, _ in names], torch.autograd.grad(y, [t for _, t in names], dy.double())))
    return out
