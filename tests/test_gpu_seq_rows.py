"""GPU: the causal sequence operators where a workgroup takes more than one row, where tensors are strided in the backward pass, and the scan
against a bound that knows how its states forget."""
import pytest
import torch

from oracle import seq
from tests.test_gpu_seq import IDS, SCAN, U, dev, leaves, ops, rnd, scan_inputs  # noqa: F401

pytestmark = pytest.mark.gpu


def near(name, got, ref, tol):
    """|got - ref| <= tol, plus the rounding to got's type; all on the device (float64)."""
    fi = torch.finfo(got.dtype)
    err = (got.detach().double() - ref).abs()
    tol = tol + fi.eps / 2 * (ref.abs() + tol) + fi.smallest_normal * fi.eps / 2
    bad = ~(err <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %.3g over a tolerance of %.3g" % (
        name, int(bad.sum()), bad.numel(), float(err[bad].max()), float(tol[bad].min()))


def top(v):
    return v.abs().amax(-1, keepdim=True)


def spaced(t, off, pitch):
    """t's values as a slice of wider rows, NaN around them."""
    wide = torch.full((t.shape[0], pitch), float("nan"), dtype=t.dtype, device=t.device)
    wide[:, off:off + t.shape[1]] = t
    return wide[:, off:off + t.shape[1]]


# Rows beyond what one turn of all workgroups takes (2048 forward, 512 backward, four rows each up to 1024 columns), by no whole turn, for every
# form: threads a row x column quads a thread, aligned and element by element.
RESIDUAL = [(8203, 12), (8203, 13), (8203, 500), (8203, 501), (8203, 1000), (2051, 1032), (2051, 1030), (2051, 4096), (2051, 4100), (2051, 4097),
            (2051, 8196), (2051, 8193)]


@pytest.mark.parametrize("dtype,wide", [(torch.float32, True), (torch.bfloat16, True), (torch.bfloat16, False)], ids=["fp32", "bf16-fp32", "bf16"])
@pytest.mark.parametrize("R,C", RESIDUAL)
def test_residual_norm_over_many_rows(ops, R, C, dtype, wide):
    g = torch.Generator(device="cuda").manual_seed(R + C)
    new = lambda *s, dt=torch.float32, std=1.0, mean=0.0: (torch.randn(s, generator=g, device="cuda") * std + mean).to(dt)     # noqa: E731
    rt = torch.float32 if wide else dtype
    x, res, w, b, s = new(R, C, dt=dtype), new(R, C, dt=rt, std=2.0), new(C, mean=1.0, std=0.3), new(C), new(C, mean=1.0)
    dy, dr = new(R, C, dt=dtype), new(R, C, dt=rt)
    k, kp = 200, 200 + 80                     # (weights' gradients: at most 5 rows a thread, 4 joined, 512 partial rows in 16 chains)
    for kind, p in (("layer", 0.3), ("rms", 0.0)):
        ins = [t.clone().requires_grad_() for t in (x, res, w, b, s)]
        y, r = ops.residual_norm(*ins, kind=kind, p=p, seed=11)
        grads = torch.autograd.grad((y, r), ins, (dy, dr))
        # the mask by the operator's own dropout, which has tests of its own; everything else in 64 bits
        kept = ops.dropout(torch.ones_like(x), p, 11).double() != 0
        xd = torch.where(kept, x.double() * seq.drop_factor(p), 0.0)
        ref = seq.residual_norm(xd, res, w, b, s, kind=kind, kept=r.detach(), dy=dy, dr=dr)
        ref["dx"] = torch.where(kept, ref["dx"] * seq.drop_factor(p), 0.0)
        near("r", r, ref["r"], 4 * U * (xd.abs() * s.double().abs() + res.double().abs()))
        kd = r.detach().double()
        v = kd - kd.mean(-1, keepdim=True) if kind == "layer" else kd
        rstd = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-5)
        hm = top(kd) * rstd
        near("y", y, ref["y"], k * U * (hm * w.double().abs() * (1 + hm * hm * (kind == "layer")) + b.double().abs()))
        gm = top(dy.double() * w.double())
        dm = rstd * gm * (2 + 2 * hm * hm) * (1 + hm * hm) + dr.double().abs()
        near("dx", grads[0], ref["dx"], k * U * dm * s.double().abs() * seq.drop_factor(p))
        near("dresidual", grads[1], ref["dresidual"], k * U * dm)
        near("dweight", grads[2], ref["dweight"], kp * U * (dy.double().abs() * hm * (1 + hm * hm)).sum(0))
        near("dbias", grads[3], ref["dbias"], 80 * U * dy.double().abs().sum(0))
        near("dscale", grads[4], ref["dscale"], kp * U * (dm * xd.abs()).sum(0))
        # strided, aligned (a pitch of whole quads) and not: the same bits
        for off, pitch in ((4, C + (-C) % 4 + 8), (3, C + 5)):
            i2 = [spaced(x, off, pitch).requires_grad_(), spaced(res, off, pitch).requires_grad_()] + ins[2:]
            y2, r2 = ops.residual_norm(*i2, kind=kind, p=p, seed=11)
            g2 = torch.autograd.grad((y2, r2), i2, (spaced(dy, off, pitch), spaced(dr, off, pitch)))
            for a, c in zip((y, r) + grads, (y2, r2) + g2):
                assert torch.equal(a, c)
    # without a residual the norm keeps x itself, at x's own pitch
    grads = None
    for off, pitch in ((0, C), (4, C + (-C) % 4 + 8), (3, C + 5)):
        a, ww = spaced(x, off, pitch).requires_grad_(), w.clone().requires_grad_()
        y, r = ops.residual_norm(a, weight=ww)
        got = (y,) + torch.autograd.grad((y, r), (a, ww), (spaced(dy, off, pitch), spaced(dy, off, pitch)))
        if grads is None:
            grads = got
            ref = seq.residual_norm(x, weight=w, dy=dy, dr=dy)
            rstd = 1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + 1e-5)
            hm, gm = top(x.double()) * rstd, top(dy.double() * w.double())
            near("y alone", y, ref["y"], k * U * hm * w.double().abs())
            near("dx alone", got[1], ref["dx"], k * U * (rstd * gm * (2 + 2 * hm * hm) * (1 + hm * hm) + dy.double().abs()))
            near("dweight alone", got[2], ref["dweight"], kp * U * (dy.double().abs() * hm * (1 + hm * hm)).sum(0))
        for u, v in zip(grads, got):
            assert torch.equal(u, v)


# (more groups, fewer workgroups a group: 2048 / groups forward, 1024 / groups backward)
GATED = [(300, 64, 12), (300, 64, 13), (523, 16, 500), (523, 16, 501), (523, 16, 1000), (131, 16, 1032), (131, 16, 1030), (131, 16, 2052),
         (131, 16, 4100), (131, 16, 4097), (131, 16, 8196), (131, 16, 8193), (4099, 1, 20), (2051, 1, 2000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("R,groups,cg", GATED)
def test_gated_norm_over_many_rows(ops, R, groups, cg, dtype):
    g = torch.Generator(device="cuda").manual_seed(R + cg)
    C = groups * cg
    new = lambda *s, dt=dtype, std=1.0, mean=0.0: (torch.randn(s, generator=g, device="cuda") * std + mean).to(dt)     # noqa: E731
    x, z, dy, w = new(R, C), new(R, C), new(R, C), new(C, dt=torch.float32, mean=1.0, std=0.3)
    per = lambda t: t.unflatten(-1, (groups, -1)).abs().amax(-1, keepdim=True).expand(R, groups, cg).flatten(-2)       # noqa: E731
    k = 220
    for first in (False, True):
        ins = [t.clone().requires_grad_() for t in (x, z, w)]
        y = ops.gated_norm(*ins, groups=groups, norm_first=first)
        grads = torch.autograd.grad(y, ins, dy)
        ref = seq.gated_norm(x, z, w, 1e-5, groups, first, dy)
        gt = z.double() * torch.sigmoid(z.double())
        v = (x.double() if first else x.double() * gt)
        rstd = (1 / torch.sqrt(v.unflatten(-1, (groups, -1)).square().mean(-1, keepdim=True) + 1e-5)).expand(R, groups, cg).flatten(-2)
        out = gt.abs() if first else 1
        hm, gm, wm = v.abs() * rstd, dy.double().abs() * w.double().abs() * out, w.double().abs()
        dvm = rstd * (gm + per(hm) * per(gm) * per(hm))
        near("y", y, ref["y"], k * U * hm * wm * out)
        near("dx", grads[0], ref["dx"], k * U * (dvm if first else dvm * gt.abs()))
        near("dgate", grads[1], ref["dgate"], k * U * 1.2 * (dy.double().abs() * hm * wm if first else dvm * x.double().abs()))
        near("dweight", grads[2], ref["dweight"], (k + 80) * U * (dy.double().abs() * hm * out).sum(0))
        for off, pitch in ((4, C + (-C) % 4 + 8), (3, C + 5)):
            i2 = [spaced(x, off, pitch).requires_grad_(), spaced(z, off, pitch).requires_grad_(), ins[2]]
            y2 = ops.gated_norm(*i2, groups=groups, norm_first=first)
            for a, c in zip((y,) + grads, (y2,) + torch.autograd.grad(y2, i2, spaced(dy, off, pitch))):
                assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=IDS.get)
def test_dropout_over_more_than_one_turn(ops, dtype):
    """More elements than one turn of all workgroups takes (2^24), aligned and not: in pieces, each with its counters, the same bits; and
    head, seam and tail against the generator."""
    n, p, seed = 2 ** 24 + 4099, 0.3, 77
    x = torch.randn(n + 1, device="cuda").to(dtype)
    for t in (x[:n], x[1:]):
        y = ops.dropout(t, p, seed)
        cut = 2 ** 23
        assert torch.equal(y, torch.cat([ops.dropout(t[a:min(a + cut, n)], p, seed, a // 8) for a in range(0, n, cut)]))
        for a in (0, 2 ** 24 - 32, n // 8 * 8 - 64):
            part = t[a:a + 67].cpu()
            keep = seq.keep_mask(part.numel(), p, seed, a // 8)
            assert torch.equal(y[a:a + 67].cpu() != 0, keep & (part != 0))


def test_scan_sums_over_more_than_one_turn(ops):
    """More gradients of B and C than one turn of the finishing launch takes (2^21)."""
    T, N, Ch, S = 700, 24, 3, 64
    i = scan_inputs(T, N, Ch, S, 1, torch.float32)
    check_scan(ops, i)


# ------------------------------------------------------------------------------------------------------------ the scan, within its memory
def scan_bound(i):
    """Bounds of the fp32 kernels' errors, to first order, carried along the recurrences: what is lost in a frame is forgotten as the states
    forget.  In units of u = 2^-24, with every term by its size (HM, GM: the recurrences on absolute values):
      d is off by 8 (softplus; exp2 and reciprocal at 2, three products, a sum); a = exp2(d A2) by |d A| (8 + 2) of itself for its argument and 2
      for the exponential - and, where the time axis is split, a chunk's sum of d adds at most 8 tiles + 16 joins to the 10;
      h: a |h| (|dA| c + 2) + |d x B| (8 + 3) + |h|;   sums over states: 4 per lane and group of 16, 3 joins;
      gate z sigmoid(z): 6 + |z| of itself."""
    x, dt, A, B, C, z, dy = (i[k].double() for k in ("x", "dt", "A", "B", "C", "z", "dy"))
    T, N, Ch = x.shape
    S, G = A.shape[1], B.shape[2]
    on = (torch.arange(T).unsqueeze(1) < i["lengths"].clamp(0, T)).unsqueeze(2).double() if i["lengths"] is not None else torch.ones(T, N, 1).double()
    d = torch.logaddexp(dt + i["b"].double(), torch.zeros_like(dt)) * on
    slope = torch.sigmoid(dt + i["b"].double())
    x, z, dy, D = x.abs() * on, z, dy.abs() * on, i["D"].double().abs()
    Bc, Cc = (v.abs().repeat_interleave(Ch // G, 2) * on.unsqueeze(3) for v in (B, C))
    sg = torch.sigmoid(z)
    gate, gsl, zk = (z * sg).abs(), sg * (1 + z.abs() * (1 - sg)), z.abs()
    ng = (S + 15) // 16
    c, ks = 10 + 8 + 16, 4 * ng + 3
    a, dA = torch.exp(d.unsqueeze(-1) * A), d.unsqueeze(-1) * A.abs()
    inp = (d * x).unsqueeze(-1) * Bc
    h, e = (i["state"].double().abs() if i.get("with_state") else torch.zeros(N, Ch, S).double()), torch.zeros(N, Ch, S).double()
    H, E, P, EP = [], [], [], []
    for t in range(T):
        p, ep = a[t] * h, a[t] * e + (dA[t] * c + 3) * a[t] * h
        h = p + inp[t]
        e = ep + 11 * inp[t] + h
        P.append(p), EP.append(ep), H.append(h), E.append(e)
    H, E, P, EP = map(torch.stack, (H, E, P, EP))
    o = (H * Cc).sum(-1) + D * x
    eo = (E * Cc).sum(-1) + ks * (H * Cc).sum(-1) + 2 * o
    out = dict(y=gate * eo + (7 + zk) * gate * o, state=e)
    go = dy * gate
    gk = (8 + zk).unsqueeze(-1)
    out["dz"] = dy * gsl * eo + (12 + zk) * dy * gsl * o
    cg, ec = torch.zeros(N, Ch, S).double(), torch.zeros(N, Ch, S).double()
    du, eu, dw, ew, gm, eg = [None] * T, [None] * T, [None] * T, [None] * T, [None] * T, [None] * T
    for t in reversed(range(T)):
        g = cg + go[t].unsqueeze(-1) * Cc[t]
        e = ec + (gk[t] + 1) * go[t].unsqueeze(-1) * Cc[t] + g
        gm[t], eg[t] = g, e
        du[t] = (g * Bc[t]).sum(-1)
        eu[t] = (e * Bc[t]).sum(-1) + ks * du[t]
        dw[t] = (g * P[t] * A.abs()).sum(-1)
        ew[t] = ((e * P[t] + g * EP[t]) * A.abs()).sum(-1) + (ks + 4) * dw[t]
        cg, ec = a[t] * g, a[t] * e + (dA[t] * c + 3) * a[t] * g
    du, eu, dw, ew, gm, eg = map(torch.stack, (du, eu, dw, ew, gm, eg))
    out["dx"] = d * eu + 11 * d * du + (10 + zk) * D * go
    out["ddt"] = slope * (ew + x * eu + 12 * (dw + x * du))
    out["ddt_bias"] = out["ddt"].sum((0, 1)) + (T + N + 40) * (slope * (dw + x * du)).sum((0, 1))
    out["dD"] = (T + N + 60) * (go * x).sum((0, 1)) + (zk * go * x).sum((0, 1))
    out["dA"] = ((P * eg + EP * gm) * d.unsqueeze(-1)).sum((0, 1)) + (T + N + 50) * (gm * P * d.unsqueeze(-1)).sum((0, 1))
    grp = lambda v: v.view(T, N, G, Ch // G, S).sum(3)     # noqa: E731
    kc = 20 + Ch // 64
    dxu = (d * x).unsqueeze(-1)
    out["dB"] = grp(eg * dxu) + (kc + 10) * grp(gm * dxu)
    out["dC"] = grp(go.unsqueeze(-1) * (E + (gk + kc) * H))
    return {k: v * U * 1.01 for k, v in out.items()}


def check_scan(ops, i):
    args = [i[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "b")]
    ref, mag = (seq.scan(*args, lengths=i["lengths"], dy=i["dy"], mag=m) for m in (False, True))
    bound = scan_bound(i)
    ins = leaves(*args)
    y = ops.ssm_scan(*ins[:5], D=ins[5], z=ins[6], dt_bias=ins[7], lengths=dev(i["lengths"]))
    y.backward(dev(i["dy"]))
    got = dict(y=y, **{n: t.grad for n, t in zip(("dx", "ddt", "dA", "dB", "dC", "dD", "dz", "ddt_bias"), ins)})
    for name, t in got.items():
        near(name, t.cpu(), ref[name], bound[name])
        if name in mag:                       # (a chain of T sums is in the parameters' bounds)
            assert float(bound[name].sum()) <= (1e-4 if name in ("dA", "dD", "ddt_bias") else 2e-5) * float(mag[name].sum()), name
    state = dev(i["state"])
    y = ops.ssm_scan(*(dev(v) for v in args[:5]), D=dev(i["D"]), z=dev(i["z"]), dt_bias=dev(i["b"]), lengths=dev(i["lengths"]), state=state)
    ref = seq.scan(*args, lengths=i["lengths"], state=i["state"])
    bound = scan_bound(dict(i, with_state=True))
    near("y over a state", y.cpu(), ref["y"], bound["y"])
    near("state", state.cpu(), ref["state"], bound["state"])


@pytest.mark.parametrize("T,N,Ch,S,G", SCAN)
def test_scan_within_what_its_states_remember(ops, T, N, Ch, S, G):
    """All results in fp32, split time axis and not.  The bound stays near 1e-5 of the terms' sizes however long the row: an operand held in
    16 bits (2^-9 to 2^-12) does not pass."""
    check_scan(ops, scan_inputs(T, N, Ch, S, G, torch.float32))
