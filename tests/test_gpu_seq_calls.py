"""GPU: calls of the causal sequence operators that their documentation allows and tests/test_gpu_seq.py does not make."""
import pytest
import torch

from oracle import seq
from tests.test_gpu_seq import IDS, U, close, dev, leaves, ops, rnd  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------------------- saved tensors
def test_saved_tensors_by_way_of_the_host(ops):
    """torch.autograd.graph.save_on_cpu hands slices and transposes back at other strides: the same gradients, bit for bit."""
    g = torch.Generator().manual_seed(1)
    T, N, C = 19, 3, 20
    wide, bc, dy = (rnd(g, T, N, n).cuda() for n in (3 * C + 4, 36, C))
    first = rnd(g, N, T, C).cuda().transpose(0, 1)
    w, A, v = rnd(g, C, 4).cuda(), -torch.ones(C, 16, device="cuda"), rnd(g, C, mean=1.0).cuda()

    def grads():
        xs, b, f = (t.detach().requires_grad_() for t in (wide, bc, first))
        ps = [t.detach().clone().requires_grad_() for t in (w, A, v)]
        x, z, e = xs[..., :C], xs[..., C:2 * C], xs[..., 2 * C + 4:]
        u = ops.causal_conv1d(x, ps[0])
        h = ops.ssm_scan(f, z, ps[1], b[..., :16], b[..., 20:], D=ps[2], z=e)
        n = ops.gated_norm(x, e, ps[2])
        y, r = ops.residual_norm(z, e, ps[2], scale=ps[2], p=0.3, seed=3)
        y2, r2 = ops.residual_norm(e, weight=ps[2])
        return torch.autograd.grad([u, h, n, y, r, y2, r2], [xs, b, f] + ps, [dy] * 7)
    plain = grads()
    with torch.autograd.graph.save_on_cpu():
        away = grads()
    for a, b in zip(plain, away):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------------- scan: the ends of the ranges
@pytest.mark.parametrize("rate", [float("-inf"), -3.2e38], ids=["infinite", "overflowing"])
def test_scan_rates_without_memory(ops, rate):
    """A = -inf (-exp of a large parameter): h = d x B of the frame alone, and what lies behind a row's end, inside its last tile too,
    leaves the state as it is."""
    T, N, Ch, S = 21, 3, 6, 5
    g = torch.Generator().manual_seed(3)
    x, dt, B, C, dy = rnd(g, T, N, Ch), rnd(g, T, N, Ch), rnd(g, T, N, S), rnd(g, T, N, S), rnd(g, T, N, Ch)
    A = torch.full((Ch, S), rate)
    n = torch.tensor([21, 2, 0], dtype=torch.int32)
    for T1 in (T, 1):                                     # (one frame is a kernel of its own)
        ref = seq.scan(x[:T1], dt[:T1], A, B[:T1], C[:T1], lengths=n, state=torch.ones(N, Ch, S))
        mag = seq.scan(x[:T1], dt[:T1], A, B[:T1], C[:T1], lengths=n, state=torch.ones(N, Ch, S), mag=True)
        state = torch.ones(N, Ch, S, device="cuda")
        y = ops.ssm_scan(*map(dev, (x[:T1], dt[:T1], A, B[:T1], C[:T1])), lengths=dev(n), state=state)
        close("y", y, ref["y"], mag["y"], S + 40)         # softplus, two products, a sum over the states
        close("state", state, ref["state"], mag["state"], 40)
    ins = leaves(x, dt, A, B, C)
    ops.ssm_scan(*ins, lengths=dev(n)).backward(dev(dy))
    finite = torch.full((Ch, S), -1e30)                   # the same decay, 0, and defined derivatives: q = g a h[t-1] is 0
    ref, mag = (seq.scan(x, dt, finite, B, C, lengths=n, dy=dy, mag=m) for m in (False, True))
    for name, t in zip(("dx", "ddt", "dB", "dC"), (ins[0], ins[1], ins[3], ins[4])):
        close(name, t.grad, ref[name].view_as(t), mag[name].view_as(t), S + Ch + 60)
    assert not ins[2].grad.any()


def test_scan_growth_before_the_signal(ops):
    """Rates above zero over a silent beginning, long enough that the time axis is split and a chunk's growth passes fp32: zeros stay
    zeros, and a small state grows to what it is."""
    T, Ch, S = 1024, 3, 4                                 # one workgroup: split into chunks of 64 frames
    d, A = 0.5, 5.0                                       # e^2.5 a frame
    x, B = torch.zeros(T, 1, Ch), torch.ones(T, 1, S)
    x[1010:] = 1.0
    dt = torch.full((T, 1, Ch), d)
    rates = torch.full((Ch, S), A)
    ref, mag = (seq.scan(x, dt, rates, B, B, softplus=False, mag=m) for m in (False, True))
    y = ops.ssm_scan(*map(dev, (x, dt, rates, B, B)), softplus=False)
    close("y", y, ref["y"], mag["y"], 14 * 8 + 20)        # per frame a few roundings of the exponent, 2.5 exp and the sum
    # backwards: the gradient of the frames behind the loss is zero, however much they would grow
    dy = torch.zeros(T, 1, Ch)
    dy[:10] = 1.0
    x = torch.zeros(T, 1, Ch)
    ref, mag = (seq.scan(x, dt, rates, B, B, softplus=False, dy=dy, mag=m) for m in (False, True))
    ins = leaves(x, dt, rates, B, B)
    ops.ssm_scan(*ins, softplus=False).backward(dev(dy))
    for name, t in zip(("dx", "ddt", "dA", "dB", "dC"), ins):
        close(name, t.grad, ref[name].view_as(t), mag[name].view_as(t), 10 * 8 + 20)


def test_scan_gradients_behind_a_row_whose_state_overflowed(ops):
    """Frames behind a row's end have zero gradients, whatever became of the row; the other rows know nothing of it."""
    T, N, Ch, S = 40, 2, 4, 3
    g = torch.Generator().manual_seed(4)
    x, dt, B, C, z, dy = (rnd(g, T, N, n) for n in (Ch, Ch, S, S, Ch, Ch))
    A = -torch.ones(Ch, S)
    n = torch.tensor([5, 40], dtype=torch.int32)
    ref = seq.scan(x[:, 1:], dt[:, 1:], A, B[:, 1:], C[:, 1:], z=z[:, 1:], dy=dy[:, 1:])
    mag = seq.scan(x[:, 1:], dt[:, 1:], A, B[:, 1:], C[:, 1:], z=z[:, 1:], dy=dy[:, 1:], mag=True)
    x[:5, 0], B[:5, 0] = 1e30, 1e30
    ins = leaves(x, dt, A, B, C)
    zz, = leaves(z)
    y = ops.ssm_scan(*ins, z=zz, lengths=dev(n))
    y.backward(dev(dy))
    assert not torch.isfinite(y[:5, 0]).all() and not y[5:, 0].any()
    for t in (ins[0], ins[1], ins[3], ins[4], zz):
        assert not t.grad[5:, 0].any()
    for name, t in (("dx", ins[0]), ("ddt", ins[1]), ("dB", ins[3]), ("dC", ins[4]), ("dz", zz)):
        close(name, t.grad[:, 1:], ref[name].view_as(t[:, 1:]), mag[name].view_as(t[:, 1:]), 2 * (T * 16 + S + 64) + Ch)


def test_scan_of_no_channels(ops):
    """B and C get gradients of zero, not what the memory held."""
    A = torch.zeros(0, 4, device="cuda", requires_grad=True)
    x = torch.zeros(3, 2, 0, device="cuda", requires_grad=True)
    B = torch.ones(3, 2, 4, device="cuda", requires_grad=True)
    C = torch.ones(3, 2, 4, device="cuda", requires_grad=True)
    for _ in range(3):
        full = torch.full((3, 2, 1, 4), 7.0, device="cuda")      # (the block that the gradients are likely to be given)
        del full
        dB, dC, dA = torch.autograd.grad(ops.ssm_scan(x, x, A, B, C), (B, C, A), torch.zeros(3, 2, 0, device="cuda"))
        assert not dB.any() and not dC.any() and dA.shape == (0, 4)


# ------------------------------------------------------------------------------------------------- norms: rows far from one in size
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=IDS.get)
@pytest.mark.parametrize("C", [12, 13, 700, 1500, 1501, 4096, 9000])
def test_norms_of_rows_whose_squares_leave_fp32(ops, C, dtype):
    """Rows of 1e-36 to 1e30 in one call, among them ordinary ones: the squares underflow (with eps = 0) or overflow, the norms do not.
    Tolerances as for ordinary rows: 200 roundings of the largest value's share."""
    sizes = [1.0, 1e-18, 1e-21, 1e-30, 1e-36, 3e18, 1e25, 1e30, 2.0]
    g = torch.Generator().manual_seed(C)
    R, k = len(sizes), 220
    scale = torch.tensor(sizes).unsqueeze(1)
    x, z, w, dy = (rnd(g, R, C) * scale).to(dtype), rnd(g, R, C, dtype=dtype), rnd(g, C, mean=1.0, std=0.3), rnd(g, R, C, dtype=dtype)
    top = lambda v: v.abs().amax(-1, keepdim=True)     # noqa: E731
    for eps in (0.0, 1e-5):
        for kind in ("rms", "layer"):
            ref = seq.residual_norm(x, weight=w, eps=eps, kind=kind, dy=dy)
            xx, ww = leaves(x, w)
            y, _ = ops.residual_norm(xx, weight=ww, eps=eps, kind=kind)
            y.backward(dev(dy))
            v = x.double()
            v = v - v.mean(-1, keepdim=True) if kind == "layer" else v
            rstd = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
            hm, gm = top(x.double()) * rstd, top(dy.double() * w.double())
            close("y", y, ref["y"], hm * w.double().abs() * (1 + hm * hm * (kind == "layer")), k)
            close("dx", xx.grad, ref["dx"], rstd * gm * (2 + 2 * hm * hm) * (1 + hm * hm), k)
            close("dw", ww.grad, ref["dweight"], (dy.double().abs() * hm * (1 + hm * hm)).sum(0), k + R)
        for first in (False, True):
            ref = seq.gated_norm(x, z, w, eps, 1, first, dy)
            xx, zz, ww = leaves(x, z, w)
            y = ops.gated_norm(xx, zz, ww, eps=eps, norm_first=first)
            y.backward(dev(dy))
            gt = z.double() * torch.sigmoid(z.double())
            v = x.double() if first else x.double() * gt
            rstd = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
            # (x silu(gate) is a product in fp32: below 2^-126 a multiple of 2^-149, off by up to 2^-150 whatever its size)
            lost = 0.0 if first else 2.0 ** -150 / (k * U)
            hm, gm, out = (v.abs() + lost) * rstd, dy.double().abs() * w.double().abs() * (gt.abs() if first else 1), gt.abs() if first else 1
            dvm = rstd * (gm + top(hm) * top(gm) * top(hm))
            close("y", y, ref["y"], hm * w.double().abs() * out, k)
            close("dx", xx.grad, ref["dx"], dvm if first else dvm * gt.abs(), k)
            close("dgate", zz.grad, ref["dgate"], dy.double().abs() * hm * w.double().abs() * 1.2 if first else dvm * x.double().abs() * 1.2, k)
            close("dw", ww.grad, ref["dweight"], (dy.double().abs() * hm * out).sum(0), k + R)


# --------------------------------------------------------------------------------------------- states in graphs, two threads, far offsets
def _stream_step(ops, p):
    def step(x, res, cs, ss):
        y, r = ops.residual_norm(x, res, p["w"])
        u = ops.causal_conv1d(y, p["cw"], state=cs)
        h = ops.ssm_scan(u, y, p["A"], y[..., :16], y[..., 4:20], D=p["w"], state=ss)
        return ops.gated_norm(h, y, p["w"]), r
    return step


def test_single_frames_and_prompts_replayed_from_graphs(ops):
    """The states are read and written in place by every replay: a frame at a time, and a prompt whose time axis is split."""
    g = torch.Generator().manual_seed(20)
    C, N = 24, 2
    p = dict(w=rnd(g, C, mean=1.0, std=0.1).cuda(), cw=rnd(g, C, 4).cuda(), A=-torch.rand(C, 16).cuda() - 0.1)
    step = _stream_step(ops, p)
    with torch.no_grad():
        for T in (1, 300):
            x, res = torch.zeros(T, N, C, device="cuda"), torch.zeros(T, N, C, device="cuda")
            cs, ss = torch.zeros(N, 3, C, device="cuda"), torch.zeros(N, C, 16, device="cuda")
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step(x, res, cs, ss)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(x, res, cs, ss)
            c2, s2 = rnd(g, N, 3, C).cuda(), rnd(g, N, C, 16).cuda()
            cs.copy_(c2)
            ss.copy_(s2)
            for _ in range(5):
                x.copy_(rnd(g, T, N, C))
                res.copy_(rnd(g, T, N, C))
                graph.replay()
                torch.cuda.synchronize()
                got = [v.clone() for v in out]
                want = step(x, res, c2, s2)
                for a, b in zip(got + [cs, ss], list(want) + [c2, s2]):
                    assert torch.equal(a, b)


def test_two_threads_on_their_own_streams(ops):
    """Each thread's training steps give what they give alone."""
    import threading

    def work(seed, stream, out):
        with torch.cuda.stream(stream):
            g = torch.Generator().manual_seed(seed)
            T, N, C = 90, 2, 40 + 8 * seed
            for _ in range(6):
                x, z, dy = (rnd(g, T, N, C).cuda().requires_grad_(i < 2) for i in range(3))
                A, B, w = (-torch.ones(C, 16)).cuda().requires_grad_(), rnd(g, T, N, 16).cuda().requires_grad_(), rnd(g, C, mean=1.0).cuda().requires_grad_()
                y = ops.ssm_scan(ops.causal_conv1d(x, rnd(g, C, 4).cuda()), z, A, B, B, z=z)
                y, r = ops.residual_norm(ops.gated_norm(y, z, w), ops.dropout(x, 0.2, seed), w, p=0.1, seed=seed)
                out.append([t.clone() for t in (y, r) + torch.autograd.grad((y, r), (x, z, A, B, w), (dy, dy))])
            stream.synchronize()
    alone, both, streams = [[], []], [[], []], [torch.cuda.Stream() for _ in range(2)]
    for k in range(2):
        work(k, streams[k], alone[k])
    threads = [threading.Thread(target=work, args=(k, streams[k], both[k])) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for k in range(2):
        assert len(both[k]) == 6
        for a, b in zip(alone[k], both[k]):
            for u, v in zip(a, b):
                assert torch.equal(u, v)


def test_rows_far_apart(ops):
    """Views whose offsets pass 2^31 elements: three frames of two rows, spread over one allocation."""
    g = torch.Generator().manual_seed(21)
    T, N, C, far, row = 3, 2, 8, 900_000_000, 400_000_000
    room = torch.empty(2 * far + row + 128, dtype=torch.bfloat16, device="cuda")

    def spread(t, at):
        v = room.as_strided(t.shape, (far, row) + t.stride()[2:], at)
        v.copy_(t)
        return v
    x, dt, z, B, dy = (rnd(g, T, N, n, dtype=torch.bfloat16).cuda() for n in (C, C, C, 16, C))
    w, A, v = rnd(g, C, 4).cuda(), -torch.ones(C, 16, device="cuda"), rnd(g, C, mean=1.0).cuda()

    def grads(x, dt, z, B, dy):
        ins = [t.detach().requires_grad_() for t in (x, dt, z, B)]
        ps = [t.detach().clone().requires_grad_() for t in (w, A, v)]
        outs = [ops.causal_conv1d(ins[0], ps[0]), ops.ssm_scan(ins[0], ins[1], ps[1], ins[3], ins[3], D=ps[2], z=ins[2])]
        rows = [ins[0][:, 0], ins[2][:, 1]]                # a row pitch of `far`
        y, r = ops.residual_norm(*rows, ps[2], scale=ps[2])
        outs += [y, r, ops.gated_norm(*rows, ps[2])]
        got = torch.autograd.grad(outs, ps, [dy, dy] + [dy[:, 0]] * 3, retain_graph=True)
        return outs + list(got)
    near = grads(x, dt, z, B, dy)
    away = grads(*(spread(t, 16 * i) for i, t in enumerate((x, dt, z, B, dy))))
    for a, b in zip(near, away):
        assert torch.equal(a, b)


def test_more_than_2_to_the_31_elements(ops):
    """Outputs past 32-bit offsets: the last rows of a large call are what they are in a small one."""
    def tail(f, n):
        whole, part = f(slice(None)), f(slice(-n, None))
        for a, b in zip(whole, part):
            a = a[-n:] if a.shape[0] != b.shape[0] else a
            assert torch.equal(a, b)
    R, C = 2 ** 21 + 5, 1032
    x = torch.randn(R, C, device="cuda", dtype=torch.bfloat16)
    w = torch.rand(C, device="cuda")
    tail(lambda s: ops.residual_norm(x[s], x[s], w), 9)
    tail(lambda s: (ops.gated_norm(x[s], x[s], w),), 9)
    off = (R - 16) * C // 8
    assert torch.equal(ops.dropout(x, 0.4, 3)[-16:], ops.dropout(x[-16:], 0.4, 3, off))
    T, N = 2 ** 16, 32
    v = x[:T * N].view(T, N, C)
    k = torch.rand(C, 4, device="cuda")
    a = ops.causal_conv1d(v, k)
    assert torch.equal(a[-20:], ops.causal_conv1d(v[-23:], k)[3:])
    del a
    # the scan, rows last: every row is on its own
    s, A = v.view(2048, 1024, C), -torch.ones(C, 4, device="cuda")
    B = torch.randn(2048, 1024, 4, device="cuda", dtype=torch.bfloat16)
    a = ops.ssm_scan(s, s, A, B, B, z=s)
    b = ops.ssm_scan(s[:, -300:], s[:, -300:], A, B[:, -300:], B[:, -300:], z=s[:, -300:])     # (enough rows to be unsplit, too)
    assert torch.equal(a[:, -300:], b)
