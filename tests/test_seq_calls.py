"""CPU (-m "not gpu"): calls of the causal sequence operators that their documentation allows, up to the library's door: host tensors pass
for device tensors and every entry point is replaced by one that writes its arguments down."""
import pytest
import torch

from aas_enhancement_amd import _lib, ops_seq


class Recorder:
    """In place of the library: entry points by name, each call's arguments kept."""

    def __init__(self):
        self.calls, self.barred = [], {}

    def __getattr__(self, name):
        def entry(*args):
            assert len(args) == len(_lib.SIGNATURES[name]), name
            if name.endswith("_ws_bytes"):
                return 64
            self.calls.append((name, args))
            given = [v for a in args for v in (ops_seq._SCAN.unpack(a) if isinstance(a, bytes) else (a,))]
            assert not set(given) & set(self.barred), name        # (while they live: an address may be another's afterwards)
            return 0
        return entry

    def args(self, name):
        return [a for n, a in self.calls if n == name][-1]


@pytest.fixture
def door(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(ops_seq, "require_cuda", lambda *t: None)
    monkeypatch.setattr(ops_seq, "_stream", lambda t: 0)
    monkeypatch.setattr(ops_seq, "lib", lambda: rec)
    return rec


class relaid:
    """Saved tensors come back contiguous, as from torch.autograd.graph.save_on_cpu; `strides` knows what lies at an address."""

    def __init__(self, order=lambda t: t.contiguous()):
        self.strides, self.kept, self.order = {}, [], order

    def __enter__(self):
        self.hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format), self.unpack)
        self.hooks.__enter__()
        return self

    def __exit__(self, *e):
        self.hooks.__exit__(*e)

    def unpack(self, t):
        t = self.order(t)
        self.kept.append(t)
        self.strides[t.data_ptr()] = t.stride()
        return t


def test_gated_norm_reads_saved_rows_where_they_lie(door):
    x, wide = torch.randn(6, 16), torch.randn(6, 24, requires_grad=True)
    w = torch.ones(8, requires_grad=True)
    with relaid() as s:
        ops_seq.gated_norm(x[:, :8], wide[:, 4:12], w).sum().backward()
    a = door.args("aas_gated_norm_bwd")
    assert s.strides[a[7]] == (8, 1) and a[8] == 8
    assert s.strides[a[9]] == (8, 1) and a[10] == 8


@pytest.mark.parametrize("full", [False, True], ids=["norm", "residual"])
def test_residual_norm_reads_saved_rows_where_they_lie(door, full):
    wide, w = torch.randn(6, 24), torch.ones(8, requires_grad=True)
    res, scale = (torch.randn(6, 8), torch.ones(8, requires_grad=True)) if full else (None, None)
    with relaid() as s:
        ops_seq.residual_norm(wide[:, 4:12], res, w, scale=scale)[0].sum().backward()
    a = door.args("aas_residual_norm_bwd")
    assert s.strides[a[9]] == (8, 1) and a[10] == 8
    if full:
        assert s.strides[a[11]] == (8, 1) and a[12] == 8


def test_saved_tensors_that_come_back_spaced_out(door):
    """A hook may also hand everything back at other strides: all is read as it lies, or copied first."""
    apart = relaid(lambda t: torch.stack([t, t], -1)[..., 0])
    door.barred = apart.strides
    x, w = torch.randn(4, 3, 8), torch.randn(8, 4, requires_grad=True)
    A, B, D = torch.randn(8, 16, requires_grad=True), torch.randn(4, 3, 16), torch.ones(8)
    n = torch.full((3,), 4, dtype=torch.int32)
    g, r, v, seed = torch.ones(4, 3, 8), torch.randn(6, 8), torch.ones(8, requires_grad=True), torch.zeros(2, dtype=torch.int64)
    with apart:
        ops_seq.causal_conv1d(x, w, D, lengths=n).backward(g)
        a = door.args("aas_causal_conv1d_bwd")
        assert a[7:9] == (24, 8) and a[14:16] == (24, 8)
        ops_seq.ssm_scan(x, x, A, B, B, D=D, z=x, dt_bias=D, lengths=n).backward(g)
        f = ops_seq._SCAN.unpack(door.args("aas_ssm_scan_bwd")[1])
        assert f[17:23] == (24, 8) * 3 and f[23:] == (48, 16, 16) * 2
        ops_seq.gated_norm(r, r, v).backward(torch.ones(6, 8))
        a = door.args("aas_gated_norm_bwd")
        assert a[6] == a[8] == a[10] == 8
        ops_seq.residual_norm(r, r, v, D, scale=v, p=0.5, seed=seed)[0].backward(torch.ones(6, 8))
        a = door.args("aas_residual_norm_bwd")
        assert a[6] == a[10] == a[12] == 8
        ops_seq.dropout(r.requires_grad_(), 0.5, seed).backward(torch.ones(6, 8))
    assert apart.strides


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64], ids=str)
def test_fp32_layers_refuse_other_types(monkeypatch, dtype):
    """What the causal operators hand out in 16 bits does not go into the layers that read fp32 (past the tensor's end)."""
    from aas_enhancement_amd import ops

    def no_launch(*a):
        raise AssertionError("launched")
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "lib", no_launch)
    monkeypatch.setattr(ops, "gemm", no_launch)
    x, w, v, f = torch.zeros(4, 2, 8, dtype=dtype), torch.zeros(8, 8), torch.zeros(8), torch.zeros(4, 2, 8)
    calls = [lambda: ops.linear_rows(x, w), lambda: ops.linear_rows(f, w.to(dtype)), lambda: ops.linear_rows(f, w, v.to(dtype)),
             lambda: ops.birnn_layer(x, w, w, w, w), lambda: ops.birnn_layer(f, w, w, w, w.to(dtype)), lambda: ops.batchnorm_rows(x, v, v, v, v),
             lambda: ops.batchnorm_rows(f, v, v.to(dtype), v, v), lambda: ops.batchnorm_eval(x, v, v, v, v), lambda: ops.leaky_relu(x, 0.1),
             lambda: ops.softmax_rows(x), lambda: ops.conv1d_cl(x, torch.zeros(3, 8, 2), None, 1), lambda: ops.conv1d_cl(f, torch.zeros(3, 8, 2), v.to(dtype), 1),
             lambda: ops.l1_sum(x, f), lambda: ops.l1_sum(f, x), lambda: ops.l1_pair(x, f, f, 1.0, 1.0, torch.zeros(2, dtype=torch.float64)),
             lambda: ops.l1_scaled(f, x, 1.0, torch.zeros(1, dtype=torch.float64)), lambda: ops.ctc_sum(x, None, None, None),
             lambda: ops.ctc_scaled(x, 0, None, 1.0), lambda: ops.layout(x, "swap01"), lambda: ops.layout_cat_nct_tnc(f, x),
             lambda: ops.layout_paired_cat(f, f, x)]
    for call in calls:
        with pytest.raises(RuntimeError, match="computes in fp32"):
            call()


def _forms(x, w, A, B, v):
    """Every operator on the given tensors: activations [4, 2, 8], weight [8, 4], A [8, 16], B [4, 2, 16], channel vector [8]."""
    state = lambda *s: torch.zeros(*s)     # noqa: E731
    return [lambda: ops_seq.causal_conv1d(x, w, v), lambda: ops_seq.causal_conv1d(x.detach(), w, v), lambda: ops_seq.causal_conv1d(x, w, v, state=state(2, 3, 8)),
            lambda: ops_seq.ssm_scan(x, x, A, B, B, D=v, z=x, dt_bias=v), lambda: ops_seq.ssm_scan(x.detach(), x.detach(), A, B.detach(), B.detach()),
            lambda: ops_seq.ssm_scan(x, x, A, B, B, state=state(2, 8, 16)), lambda: ops_seq.residual_norm(x), lambda: ops_seq.residual_norm(x.detach(), x, v),
            lambda: ops_seq.residual_norm(x.detach(), x.detach(), scale=v), lambda: ops_seq.gated_norm(x, x, v), lambda: ops_seq.gated_norm(x.detach(), x),
            lambda: ops_seq.dropout(x, 0.5, 1)]


def test_forward_mode_derivatives_are_refused(door):
    """A dual tensor's tangent is not dropped without a word - with gradients wanted, without, and in a backward pass."""
    from torch.autograd import forward_ad as fw
    shapes = [(4, 2, 8), (8, 4), (8, 16), (4, 2, 16), (8,)]
    plain = [torch.randn(s) for s in shapes]
    with fw.dual_level():
        for f in _forms(*plain):
            f()                                           # (no tangents: nothing to refuse)
        dual = [fw.make_dual(t, torch.ones_like(t)) for t in plain]
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for f in _forms(*dual):
                    with pytest.raises(NotImplementedError):
                        f()
        leaf = [t.clone().requires_grad_() for t in plain]
        for f in _forms(*leaf):
            try:
                y = f()
            except RuntimeError as e:                     # (states are for inference)
                assert "inference" in str(e)
                continue
            y = y[0] if isinstance(y, tuple) else y
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, [t for t in leaf if t.requires_grad], fw.make_dual(torch.ones_like(y), torch.ones_like(y)), allow_unused=True)


def _refuses(rc, text):
    assert rc == 1 and text in _lib.lib().aas_last_error(), (rc, _lib.lib().aas_last_error())


def test_gated_norm_c_entry_refuses_a_gradient_launch_past_2_to_the_32():
    """Before anything is launched (no rows: nothing would run but the sums of nothing)."""
    one = 4096      # (never read)
    L = _lib.lib()
    _refuses(L.aas_gated_norm_bwd(None, 0, 0, 16384 * 16384, 16384, one, 8, one, 8, one, 8, None, 1e-5, 0, one, one, one, None), b"too large")


def test_gated_norm_c_entry_refuses_rows_times_groups_past_64_bits():
    one = 4096      # (never read: pointers that are missing end the calls in any case)
    L = _lib.lib()
    _refuses(L.aas_gated_norm_fwd(None, 0, 1 << 62, 16, 4, None, 16, one, 16, None, 1e-5, 0, one), b"too large")
    _refuses(L.aas_gated_norm_bwd(None, 0, 1 << 62, 16, 4, None, 16, one, 16, one, 16, None, 1e-5, 0, one, one, None, None), b"too large")


def test_norms_refuse_eps_outside_the_numbers_it_may_be(door):
    """A negative one makes the root of a negative number, a NaN or an infinite one wipes every row out."""
    x = torch.randn(4, 8)
    for eps in (-1e-5, float("nan"), float("inf")):
        for f in (lambda: ops_seq.residual_norm(x, eps=eps), lambda: ops_seq.gated_norm(x, x, eps=eps)):
            with pytest.raises(RuntimeError, match="eps must be"):
                f()
    for eps in (0.0, 0, 1e-12, 1.0):
        ops_seq.residual_norm(x, eps=eps)
        ops_seq.gated_norm(x, x, eps=eps)
    one, L = 4096, _lib.lib()      # (pointers that are missing end the calls in any case)
    for eps in (-1e-5, float("nan"), float("inf")):
        _refuses(L.aas_residual_norm_fwd(None, 0, 0, 1, 8, None, 8, None, 0, None, None, None, eps, 0, 0, 0, 0, None, None, one, one, None), b"eps")
        _refuses(L.aas_gated_norm_fwd(None, 0, 1, 8, 1, None, 8, one, 8, None, eps, 0, one), b"eps")
        _refuses(L.aas_gated_norm_bwd(None, 0, 1, 8, 1, None, 8, one, 8, one, 8, None, eps, 0, one, one, None, None), b"eps")
