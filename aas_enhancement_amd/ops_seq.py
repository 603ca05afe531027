"""Causal sequence operators: short depthwise convolution, selective state space scan, residual norm, gated norm, dropout - the parts
of a causal residual block, for a network that has to answer frame by frame (the recurrent layers of `ops` read the whole utterance).

Activations are time-major [T, N, C] (or rows [..., C] for the norms and dropout) in fp32, bf16 or fp16 and may be views - a slice of a
wider projection, a transposed [N, T, C] - as long as the channels are contiguous; anything else is copied.  Parameters, the scan's
state and every sum are fp32, the convolution's state is of x's type.  `lengths` (int32 [N] on the device, values brought into [0, T])
are the frames of each row of a padded batch: what lies behind them is not read, its outputs and gradients are zero.  Every call
launches on the current stream of its tensors' device, may be captured into a graph, and gives the same bits on every run.  First
derivatives in reverse mode only; others raise.  Names stand in `ops`: `ops.ssm_scan(...)`.
"""
import functools
import math
import struct

import torch
from torch.autograd import forward_ad as _fw

from ._lib import check, lib, ptr, require_cuda

_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # include/aas_hip.h: AAS_DT_*

_raw_stream = torch._C._cuda_getCurrentRawStream     # what torch.cuda.current_stream().cuda_stream ends in, without the object (3-6 us a call)
_empty = torch.empty
_INF = math.inf

# include/aas_hip.h: aasScan, as packed bytes (a ctypes.Structure of 36 fields takes 3 us longer to fill)
_SCAN_FIELDS = (["size", "dtype", "T", "N", "Ch", "S", "G", "softplus"], ["x", "dt", "z", "B", "C", "A", "D", "dt_bias", "len"],
                ["x_st", "x_sn", "dt_st", "dt_sn", "z_st", "z_sn", "B_st", "B_sn", "B_sg", "C_st", "C_sn", "C_sg"])
_SCAN = struct.Struct("@%di%dP%dq" % tuple(len(f) for f in _SCAN_FIELDS))


def _on_device(fn):
    """Run with the device of the first argument current (a call on a tensor of another device than the current one)."""
    @functools.wraps(fn)
    def wrapped(x, *a, **k):
        if isinstance(x, torch.Tensor) and x.is_cuda and x.get_device() != torch.cuda.current_device():
            with torch.cuda.device(x.device):
                return fn(x, *a, **k)
        return fn(x, *a, **k)
    return wrapped


def _stream(t):
    return _raw_stream(t.get_device())


class _NoSecond(torch.autograd.Function):
    """Hands a gradient on and refuses to be differentiated."""

    @staticmethod
    def forward(ctx, g, *anchors):
        return g.view_as(g)

    @staticmethod
    def backward(ctx, *g):
        raise RuntimeError("the causal sequence operators have first derivatives only: cannot differentiate through their gradients")


def _first_order(backward):
    """The backward passes are kernels without gradients of their own.  A recorded pass (create_graph=True) hands out gradients that
    refuse to be differentiated wherever they depend on something that wants a gradient."""
    @functools.wraps(backward)
    def wrapped(ctx, *g):
        if _fw._current_level >= 0:
            _no_tangents(*g, *ctx.saved_tensors)
        if not torch.is_grad_enabled():
            return backward(ctx, *g)
        with torch.no_grad():
            out = backward(ctx, *g)
        anchors = [t for t in (*ctx.saved_tensors, *g) if t is not None and t.requires_grad]
        one = lambda o: o if o is None or not anchors else _NoSecond.apply(o, *anchors)   # noqa: E731
        return tuple(one(o) for o in out)
    return wrapped


def _ws(nbytes, dev):
    return _empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _bad(who, what):
    raise RuntimeError("%s: %s" % (who, what))


def _activation(who, name, t, like=None, shape=None):
    """Checks of one activation; its channels made contiguous."""
    if like is not None and isinstance(t, torch.Tensor) and t.dtype is like.dtype and t.device == like.device and t.shape == shape and t.stride(-1) == 1:
        return t
    if not isinstance(t, torch.Tensor):
        _bad(who, "%s must be a tensor, got %s" % (name, type(t).__name__))
    require_cuda(t)
    if t.dtype not in _DT:
        _bad(who, "%s is %s; fp32, bf16 and fp16 are supported" % (name, t.dtype))
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        _bad(who, "%s is %s on %s, expected %s on %s" % (name, t.dtype, t.device, like.dtype, like.device))
    if shape is not None and tuple(t.shape) != tuple(shape):
        _bad(who, "%s has shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))
    return t if t.dim() == 0 or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _param(who, name, t, like, shape):
    """An fp32 parameter of the given shape, contiguous; None stays None."""
    if t is None or (t.dtype is torch.float32 and t.device == like.device and t.shape == shape and t.is_contiguous()):
        return t
    require_cuda(t)
    if t.dtype != torch.float32 or t.device != like.device or tuple(t.shape) != tuple(shape):
        _bad(who, "%s must be fp32 %s on %s, got %s %s on %s" % (name, tuple(shape), like.device, t.dtype, tuple(t.shape), t.device))
    return t if t.is_contiguous() else t.contiguous()


def _lengths(who, t, like, N):
    if t is None or (t.dtype is torch.int32 and t.shape == (N,) and t.device == like.device and t.is_contiguous()):
        return t
    require_cuda(t)
    if t.dtype != torch.int32 or tuple(t.shape) != (N,) or t.device != like.device:
        _bad(who, "lengths must be int32 [%d] on %s, got %s %s on %s" % (N, like.device, t.dtype, tuple(t.shape), t.device))
    return t if t.is_contiguous() else t.contiguous()


def _state(who, t, like, dtype, shape, given):
    """The in-out state: written in place, so it must be what it says, and no gradient flows through it."""
    if t is None:
        return
    require_cuda(t)
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or t.device != like.device or not t.is_contiguous():
        _bad(who, "state must be contiguous %s %s on %s, got %s %s%s on %s"
             % (dtype, tuple(shape), like.device, t.dtype, tuple(t.shape), "" if t.is_contiguous() else " (strided)", t.device))
    if _wants_grad(t, *given):
        _bad(who, "state= is for inference (under torch.no_grad() or on tensors without gradients): no gradient flows through it")


def _written(state):
    if not state.is_inference():     # (tensors made under inference_mode have no version to raise)
        torch.autograd.graph.increment_version(state)


def _no_tangents(*ts):
    """Inside a torch.autograd.forward_ad level: the kernels would hand the values on and drop the tangents."""
    for t in ts:
        if isinstance(t, torch.Tensor) and _fw.unpack_dual(t).tangent is not None:
            raise NotImplementedError("the causal sequence operators have no forward-mode derivatives")


def _wants_grad(*ts):
    if _fw._current_level >= 0:
        _no_tangents(*ts)
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


# The backward passes ask for the layouts of what they read again: what a saved-tensor hook hands back
# (torch.autograd.graph.save_on_cpu) holds the values that were saved, not their strides.
def _unit(t):
    """An activation with its channels side by side."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _whole(*ts):
    """Parameters, statistics and states, contiguous."""
    return [t if t is None or t.is_contiguous() else t.contiguous() for t in ts]


def _rows(t):
    """-> (tensor, row pitch): the leading dimensions as uniformly spaced rows, copied where they are not."""
    if t.is_contiguous():
        return t, t.shape[-1]
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        return t.contiguous(), t.shape[-1]
    pitch, seen = None, 1
    for size, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if pitch is None:
            pitch = st
        elif st != pitch * seen:
            t = t.contiguous()
            return t, t.shape[-1]
        seen *= size
    return t, t.shape[-1] if pitch is None else pitch


# ------------------------------------------------------------------------------------------------------------- causal convolution
def _conv_fwd(x, weight, bias, silu, lengths, state):
    T, N, C = x.shape
    y = _empty((T, N, C), device=x.device, dtype=x.dtype)
    check(lib().aas_causal_conv1d_fwd(_stream(x), _DT[x.dtype], T, N, C, weight.shape[1], x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(),
                                      ptr(bias), silu, ptr(lengths), ptr(state), y.data_ptr()), "aas_causal_conv1d_fwd")
    return y


class _CausalConv1d(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, silu, lengths):
        ctx.save_for_backward(x, weight, bias, lengths)
        ctx.silu = silu
        return _conv_fwd(x, weight, bias, silu, lengths, None)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, weight, bias, lengths = ctx.saved_tensors
        x, dy = _unit(x), _unit(dy)
        weight, bias, lengths = _whole(weight, bias, lengths)
        T, N, C = x.shape
        K = weight.shape[1]
        need = ctx.needs_input_grad
        dx = _empty((T, N, C), device=x.device, dtype=x.dtype) if need[0] else None
        dw = torch.empty_like(weight) if need[1] else None
        db = torch.empty_like(bias) if need[2] else None
        ws = _ws(lib().aas_causal_conv1d_bwd_ws_bytes(T, N, C, K), x.device) if need[1] or need[2] else None
        check(lib().aas_causal_conv1d_bwd(_stream(x), _DT[x.dtype], T, N, C, K, x.data_ptr(), x.stride(0), x.stride(1), weight.data_ptr(), ptr(bias),
                                          ctx.silu, ptr(lengths), dy.data_ptr(), dy.stride(0), dy.stride(1), ptr(dx), ptr(dw), ptr(db), ptr(ws)),
              "aas_causal_conv1d_bwd")
        return dx, dw, db, None, None


@_on_device
def causal_conv1d(x, weight, bias=None, activation="silu", lengths=None, state=None):
    """Depthwise causal convolution over K = 2, 3 or 4 frames: p[t] = bias + sum_k weight[:, k] x[t - K + 1 + k], y = silu(p) or p
    (activation "silu" | "none").  x [T, N, C], weight fp32 [C, K], bias fp32 [C].  state [N, K-1, C] of x's type: the frames in front of the
    first, oldest first; replaced in place by the last K-1 frames seen, so that a stream goes on call by call (T = 1 and up; inference
    only).  Without it the sequence begins with zeros; gradients for x, weight and bias."""
    who = "causal_conv1d"
    x = _activation(who, "x", x)
    if x.dim() != 3:
        _bad(who, "x must be [T, N, C], got %s" % (tuple(x.shape),))
    if activation not in ("silu", "none"):
        _bad(who, "activation must be 'silu' or 'none', got %r" % (activation,))
    N, C = x.shape[1], x.shape[2]
    if weight.dim() != 2 or not 2 <= weight.shape[1] <= 4:
        _bad(who, "weight must be [C, K] with K = 2, 3 or 4, got %s" % (tuple(weight.shape),))
    weight = _param(who, "weight", weight, x, (C, weight.shape[1]))
    bias = _param(who, "bias", bias, x, (C,))
    lengths = _lengths(who, lengths, x, N)
    silu = 1 if activation == "silu" else 0
    if state is not None:
        _state(who, state, x, x.dtype, (N, weight.shape[1] - 1, C), (x, weight, bias))
        y = _conv_fwd(x, weight, bias, silu, lengths, state)
        _written(state)
        return y
    if _wants_grad(x, weight, bias):
        return _CausalConv1d.apply(x, weight, bias, silu, lengths)
    return _conv_fwd(x, weight, bias, silu, lengths, None)


# ------------------------------------------------------------------------------------------------------------------------ the scan
def _scan_desc(x, dt, A, B, C, D, z, dt_bias, softplus, lengths):
    T, N, Ch = x.shape
    xs, ds, bs, cs = x.stride(), dt.stride(), B.stride(), C.stride()
    zs = xs if z is None else z.stride()
    p = lambda t: 0 if t is None else t.data_ptr()     # noqa: E731
    return _SCAN.pack(_SCAN.size, _DT[x.dtype], T, N, Ch, A.shape[1], B.shape[2], softplus,
                      x.data_ptr(), dt.data_ptr(), p(z), B.data_ptr(), C.data_ptr(), A.data_ptr(), p(D), p(dt_bias), p(lengths),
                      xs[0], xs[1], ds[0], ds[1], zs[0], zs[1], bs[0], bs[1], bs[2], cs[0], cs[1], cs[2])


def _scan_fwd(x, dt, A, B, C, D, z, dt_bias, softplus, lengths, state, keep):
    T, N, Ch = x.shape
    S = A.shape[1]
    y = _empty((T, N, Ch), device=x.device, dtype=x.dtype)
    hsave = _empty((2 * ((T + 15) // 16), N, Ch, S), device=x.device, dtype=torch.float32) if keep else None
    ws = None if T == 1 else _ws(lib().aas_ssm_scan_fwd_ws_bytes(T, N, Ch, S, B.shape[2]), x.device)
    d = _scan_desc(x, dt, A, B, C, D, z, dt_bias, softplus, lengths)
    check(lib().aas_ssm_scan_fwd(_stream(x), d, ptr(state), y.data_ptr(), ptr(hsave), ptr(ws)), "aas_ssm_scan_fwd")
    return y, hsave


class _SsmScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, softplus, lengths):
        y, hsave = _scan_fwd(x, dt, A, B, C, D, z, dt_bias, softplus, lengths, None, True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, lengths, hsave)
        ctx.softplus = softplus
        return y

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, dt, A, B, C, D, z, dt_bias, lengths, hsave = ctx.saved_tensors
        x, dt, B, C, z, dy = map(_unit, (x, dt, B, C, z, dy))
        A, D, dt_bias, lengths, hsave = _whole(A, D, dt_bias, lengths, hsave)
        T, N, Ch = x.shape
        S, G = A.shape[1], B.shape[2]
        dx, ddt = x.new_empty((T, N, Ch)), x.new_empty((T, N, Ch))
        dz = None if z is None else x.new_empty((T, N, Ch))
        dB, dC, dA = x.new_empty((T, N, G, S)), x.new_empty((T, N, G, S)), A.new_empty((Ch, S))
        dD = None if D is None else A.new_empty((Ch,))
        dbias = None if dt_bias is None else A.new_empty((Ch,))
        ws = _ws(lib().aas_ssm_scan_bwd_ws_bytes(T, N, Ch, S, G), x.device)
        d = _scan_desc(x, dt, A, B, C, D, z, dt_bias, ctx.softplus, lengths)
        check(lib().aas_ssm_scan_bwd(_stream(x), d, dy.data_ptr(), dy.stride(0), dy.stride(1), hsave.data_ptr(), dx.data_ptr(),
                                     ddt.data_ptr(), ptr(dz), dB.data_ptr(), dC.data_ptr(), dA.data_ptr(), ptr(dD), ptr(dbias), ptr(ws)),
              "aas_ssm_scan_bwd")
        return dx, ddt, dA, dB, dC, dD, dz, dbias, None, None


@_on_device
def ssm_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, lengths=None, state=None):
    """Selective state space scan, per row and channel over S <= 64 states:
        d[t] = softplus(dt[t] + dt_bias)   (softplus=False: the sum itself)
        h[t] = exp(d[t] A) h[t-1] + d[t] x[t] B[t],   y[t] = (C[t] . h[t] + D x[t]) silu(z[t])   (z None: no gate)
    x, dt, z [T, N, Ch]; B, C [T, N, S] or [T, N, G, S] (channel c reads group c // (Ch / G)); all of one type.  A fp32 [Ch, S], D and dt_bias
    fp32 [Ch].  state fp32 [N, Ch, S]: h in front of the first frame, replaced in place by h behind each row's last one, so that a
    prompt is read in one call and single frames (T = 1) go on from it (inference only).  Without it h starts at zero; gradients for
    every tensor, the backward pass forming h again from the states kept in front of every 8th frame (T N Ch S / 2 bytes, held from the
    forward pass on: 8 bytes an element at 16 states)."""
    who = "ssm_scan"
    x = _activation(who, "x", x)
    if x.dim() != 3:
        _bad(who, "x must be [T, N, C], got %s" % (tuple(x.shape),))
    T, N, Ch = x.shape
    if A.dim() != 2 or not 1 <= A.shape[1] <= 64:
        _bad(who, "A must be [C, S] with 1 <= S <= 64, got %s" % (tuple(A.shape),))
    S = A.shape[1]
    dt = _activation(who, "dt", dt, x, x.shape)
    if z is not None:
        z = _activation(who, "z", z, x, x.shape)
    if not isinstance(B, torch.Tensor) or not isinstance(C, torch.Tensor) or B.dim() not in (3, 4) or B.dim() != C.dim():
        _bad(who, "B and C must both be [T, N, S] or [T, N, G, S]")
    if B.dim() == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    G = B.shape[2]
    if G < 1 or Ch % G:
        _bad(who, "%d channels do not divide into the %d groups of B and C" % (Ch, G))
    B = _activation(who, "B", B, x, (T, N, G, S))
    C = _activation(who, "C", C, x, (T, N, G, S))
    A = _param(who, "A", A, x, (Ch, S))
    D = _param(who, "D", D, x, (Ch,))
    dt_bias = _param(who, "dt_bias", dt_bias, x, (Ch,))
    lengths = _lengths(who, lengths, x, N)
    softplus = 1 if softplus else 0
    if state is not None:
        _state(who, state, x, torch.float32, (N, Ch, S), (x, dt, A, B, C, D, z, dt_bias))
        y = _scan_fwd(x, dt, A, B, C, D, z, dt_bias, softplus, lengths, state, False)[0]
        _written(state)
        return y
    if _wants_grad(x, dt, A, B, C, D, z, dt_bias):
        return _SsmScan.apply(x, dt, A, B, C, D, z, dt_bias, softplus, lengths)
    return _scan_fwd(x, dt, A, B, C, D, z, dt_bias, softplus, lengths, None, False)[0]


# ------------------------------------------------------------------------------------------------------------------------- dropout
def dropout_counters(numel):
    """Counters that dropout over `numel` elements uses: two calls under one seed draw apart when their offsets differ by this much."""
    return (int(numel) + 7) // 8


def _drop_args(who, x, p, seed, offset):
    """-> (thr, seed, offset, device seed or None, buffer for the seed used or None)"""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        _bad(who, "p must be in [0, 1], got %r" % (p,))
    thr = int(math.floor(p * 65536 + 0.5))
    if thr == 0:
        return 0, 0, 0, None, None
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 2 or seed.device != x.device or not seed.is_contiguous():
            _bad(who, "a seed tensor must be int64 {seed, offset} on %s" % (x.device,))
        if offset:
            _bad(who, "the offset is part of a seed tensor")
        return thr, 0, 0, seed, torch.empty_like(seed)
    if seed is None or isinstance(seed, float):
        _bad(who, "p > 0 needs a seed (an int, or an int64 tensor {seed, offset} on the device)")
    wrap = lambda v: (int(v) + 2 ** 63) % 2 ** 64 - 2 ** 63     # noqa: E731  (64 bits, as the C side takes them)
    return thr, wrap(seed), wrap(offset), None, None


def _dropout_call(x, drop, seed_dev, used):
    y = torch.empty_like(x)
    check(lib().aas_dropout(_stream(x), _DT[x.dtype], x.numel(), x.data_ptr(), y.data_ptr(), drop[0], drop[1], drop[2], ptr(seed_dev), ptr(used)),
          "aas_dropout")
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, drop):
        ctx.drop = drop[:3]
        ctx.save_for_backward(drop[4])
        return _dropout_call(x, drop, drop[3], drop[4])

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        used, = _whole(*ctx.saved_tensors)
        return _dropout_call(dy.contiguous(), ctx.drop, used, None), None


@_on_device
def dropout(x, p, seed, offset=0):
    """x / (1 - p) where an element is kept, 0 where it is not; p is met to 2^-17.  The mask is a function of (seed, offset, element
    number) - 16 bits of Philox-4x32-10 each - and never stored: the backward pass forms it again.  seed: an int with `offset` in counters
    (`dropout_counters`), or an int64 tensor {seed, offset} on the device, read when the launch runs - a captured graph draws a new
    mask on every replay if the program advances the tensor; the backward pass uses what its forward pass read."""
    who = "dropout"
    x = _activation(who, "x", x).contiguous()
    drop = _drop_args(who, x, p, seed, offset)
    if _wants_grad(x):
        return _Dropout.apply(x, drop)
    return _dropout_call(x, drop, drop[3], None)


# ----------------------------------------------------------------------------------------------------------------------- row norms
def _res_fwd(x, x_ld, residual, res_ld, weight, bias, scale, eps, layer, drop, want_r, want_stat):
    C = x.shape[-1]
    R = x.numel() // C
    rt = x.dtype if residual is None else residual.dtype
    y = _empty(x.shape, device=x.device, dtype=x.dtype)
    r = _empty(x.shape, device=x.device, dtype=rt) if want_r else None
    stat = _empty((R, 2), device=x.device, dtype=torch.float32) if want_stat else None
    check(lib().aas_residual_norm_fwd(_stream(x), _DT[x.dtype], _DT[rt], R, C, x.data_ptr(), x_ld, ptr(residual), res_ld, ptr(weight), ptr(bias),
                                      ptr(scale), eps, layer, drop[0], drop[1], drop[2], ptr(drop[3]), ptr(drop[4]), y.data_ptr(), ptr(r),
                                      ptr(stat)), "aas_residual_norm_fwd")
    return y, r, stat


def _res_bwd(ctx, dy, dr):
    kept, x, weight, scale, stat, used = ctx.saved_tensors
    kept, kept_ld = _rows(kept)
    x, x_ld = (None, 0) if x is None else _rows(x)
    weight, scale, stat, used = _whole(weight, scale, stat, used)
    need, drop = ctx.needs_input_grad, ctx.drop
    C = kept.shape[-1]
    R = kept.numel() // C
    dev, shape = kept.device, kept.shape
    args = []
    for g in (dy, dr):
        if g is None:
            args += [None, 0]
        else:
            args += _rows(g)
    dx = _empty(shape, device=dev, dtype=ctx.x_dtype) if need[0] else None
    dres = _empty(shape, device=dev, dtype=kept.dtype) if need[1] else None
    dw, db, ds = (_empty(C, device=dev, dtype=torch.float32) if n else None for n in need[2:5])
    ws = _ws(lib().aas_residual_norm_bwd_ws_bytes(R, C), dev) if need[2] or need[3] or need[4] else None
    check(lib().aas_residual_norm_bwd(_stream(kept), _DT[ctx.x_dtype], _DT[kept.dtype], R, C, ptr(args[0]), args[1], ptr(args[2]), args[3], kept.data_ptr(),
                                      kept_ld, ptr(x), x_ld, stat.data_ptr(), ptr(weight), ptr(scale), ctx.layer, drop[0], drop[1],
                                      drop[2], ptr(used), ptr(dx), ptr(dres), ptr(dw), ptr(db), ptr(ds), ptr(ws)), "aas_residual_norm_bwd")
    return dx, dres, dw, db, ds, None, None, None


class _ResidualNorm(torch.autograd.Function):
    """(y, r) with r a tensor of its own."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, scale, eps, layer, drop):
        x, x_ld = _rows(x)
        res, res_ld = (None, 0) if residual is None else _rows(residual)
        y, r, stat = _res_fwd(x, x_ld, res, res_ld, weight, bias, scale, eps, layer, drop, True, True)
        ctx.save_for_backward(r, x if ctx.needs_input_grad[4] else None, weight, scale, stat, drop[4])
        ctx.x_dtype, ctx.layer, ctx.drop = x.dtype, layer, drop[:3]
        ctx.set_materialize_grads(False)
        return y, r

    @staticmethod
    @_first_order
    def backward(ctx, dy, dr):
        if dy is None and dr is None:
            return (None,) * 8
        return _res_bwd(ctx, dy, dr)


class _Norm(torch.autograd.Function):
    """(y, r) where nothing is added and r is x itself: handed through, so that r's gradient joins in the backward kernel instead of in a
    second sum behind a rounding."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, scale, eps, layer, drop):
        xr, x_ld = _rows(x)
        y, _, stat = _res_fwd(xr, x_ld, None, 0, weight, bias, None, eps, layer, drop, False, True)
        ctx.save_for_backward(xr, None, weight, None, stat, None)
        ctx.x_dtype, ctx.layer, ctx.drop = x.dtype, layer, drop[:3]
        ctx.set_materialize_grads(False)
        return y, x

    backward = _ResidualNorm.backward


@_on_device
def residual_norm(x, residual=None, weight=None, bias=None, scale=None, eps=1e-5, kind="rms", p=0.0, seed=None, offset=0):
    """-> (y, r): the residual sum behind a block and the norm in front of the next one, in one pass over rows of C <= 16384 channels:
        r = residual + scale * dropout(x),   y = norm(r) weight + bias,   norm "rms" (v / sqrt(mean(v^2) + eps)) or "layer" (v less its mean)
    x [..., C]; residual [..., C] of x's type or fp32 (r and its gradient are of its type; y is of x's); weight, bias, scale fp32 [C] or None.
    The norm reads r as it is kept.  Without residual, scale and dropout r is x itself.  p, seed, offset: as `dropout`, over x's elements
    in row-major order.  Gradients for all five tensors."""
    who = "residual_norm"
    x = _activation(who, "x", x)
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] > 16384:
        _bad(who, "x must be [..., C] with 1 <= C <= 16384, got %s" % (tuple(x.shape),))
    if kind not in ("rms", "layer"):
        _bad(who, "kind must be 'rms' or 'layer', got %r" % (kind,))
    C = x.shape[-1]
    if residual is not None:
        if residual.dtype not in (x.dtype, torch.float32) or residual.device != x.device or residual.shape != x.shape:
            _bad(who, "residual must be %s or fp32 %s on %s, got %s %s on %s"
                 % (x.dtype, tuple(x.shape), x.device, residual.dtype, tuple(residual.shape), residual.device))
        residual = _activation(who, "residual", residual)
    weight, bias, scale = (_param(who, n, t, x, (C,)) for n, t in (("weight", weight), ("bias", bias), ("scale", scale)))
    drop = _drop_args(who, x, p, seed, offset)
    eps, layer = float(eps), 1 if kind == "layer" else 0
    if not 0.0 <= eps < _INF:
        _bad(who, "eps must be a number from 0 on, got %r" % (eps,))
    if residual is None and scale is None and not drop[0]:
        if _wants_grad(x, weight, bias):
            return _Norm.apply(x, None, weight, bias, None, eps, layer, drop)
        xr, ld = _rows(x)
        return _res_fwd(xr, ld, None, 0, weight, bias, None, eps, layer, drop, False, False)[0], x
    if _wants_grad(x, residual, weight, bias, scale):
        return _ResidualNorm.apply(x, residual, weight, bias, scale, eps, layer, drop)
    xr, ld = _rows(x)
    rr, rld = (None, 0) if residual is None else _rows(residual)
    return _res_fwd(xr, ld, rr, rld, weight, bias, scale, eps, layer, drop, True, False)[:2]


def _gated_fwd(x, x_ld, gate, gate_ld, weight, eps, groups, norm_first):
    C = x.shape[-1]
    y = _empty(x.shape, device=x.device, dtype=x.dtype)
    check(lib().aas_gated_norm_fwd(_stream(x), _DT[x.dtype], x.numel() // C, C, groups, x.data_ptr(), x_ld, gate.data_ptr(), gate_ld, ptr(weight), eps,
                                   norm_first, y.data_ptr()), "aas_gated_norm_fwd")
    return y


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, weight, eps, groups, norm_first):
        (x, x_ld), (gate, gate_ld) = _rows(x), _rows(gate)
        ctx.save_for_backward(x, gate, weight)
        ctx.args = (eps, groups, norm_first)
        return _gated_fwd(x, x_ld, gate, gate_ld, weight, eps, groups, norm_first)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        x, gate, weight = ctx.saved_tensors
        eps, groups, norm_first = ctx.args
        (x, x_ld), (gate, gate_ld), (dy, dy_ld), (weight,) = _rows(x), _rows(gate), _rows(dy), _whole(weight)
        C = x.shape[-1]
        R = x.numel() // C
        need = ctx.needs_input_grad
        dx, dg = (_empty(x.shape, device=x.device, dtype=x.dtype) if n else None for n in need[:2])
        dw = torch.empty_like(weight) if need[2] else None
        ws = _ws(lib().aas_gated_norm_bwd_ws_bytes(R, C, groups), x.device) if need[2] else None
        check(lib().aas_gated_norm_bwd(_stream(x), _DT[x.dtype], R, C, groups, dy.data_ptr(), dy_ld, x.data_ptr(), x_ld, gate.data_ptr(), gate_ld,
                                       ptr(weight), eps, norm_first, ptr(dx), ptr(dg), ptr(dw), ptr(ws)), "aas_gated_norm_bwd")
        return dx, dg, dw, None, None, None


@_on_device
def gated_norm(x, gate, weight=None, eps=1e-5, groups=1, norm_first=False):
    """Root-mean-square norm behind a block, fused with its gate, over each of `groups` equal runs of the channels:
        norm_first=False: norm(x silu(gate)) weight;   norm_first=True: norm(x) weight silu(gate).
    x, gate [..., C] of one type (either may be a slice of a wider projection), weight fp32 [C] or None, at most 16384 channels a group.
    Gradients for all three."""
    who = "gated_norm"
    x = _activation(who, "x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        _bad(who, "x must be [..., C], got %s" % (tuple(x.shape),))
    gate = _activation(who, "gate", gate, x, x.shape)
    C, groups = x.shape[-1], int(groups)
    if groups < 1 or C % groups or C // groups > 16384:
        _bad(who, "%d channels do not divide into %d groups of at most 16384" % (C, groups))
    weight = _param(who, "weight", weight, x, (C,))
    eps, norm_first = float(eps), 1 if norm_first else 0
    if not 0.0 <= eps < _INF:
        _bad(who, "eps must be a number from 0 on, got %r" % (eps,))
    if _wants_grad(x, gate, weight):
        return _GatedNorm.apply(x, gate, weight, eps, groups, norm_first)
    (xr, x_ld), (gr, g_ld) = _rows(x), _rows(gate)
    return _gated_fwd(xr, x_ld, gr, g_ld, weight, eps, groups, norm_first)
