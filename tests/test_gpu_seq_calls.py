"""GPU: calls of the causal sequence operators that their documentation allows and tests/test_gpu_seq.py does not make."""
import pytest
import torch

from tests.test_gpu_seq import ops, rnd  # noqa: F401

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
