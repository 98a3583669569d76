"""The delta rule on heads that lie apart: head-major tensors of any length, and gradients in layouts that the kernels do not take."""
import pytest
import torch

from delta_oracle import inputs
from ray_oracle import ray_set

pytestmark = pytest.mark.gpu


def _apart(t):
    """t [n, heads, ..] with each head's rows together."""
    return t.transpose(0, 1).contiguous().transpose(0, 1)


@pytest.mark.parametrize("lens", [[28] * 5001, [1] * 140000, [3, 0] * 47000])
def test_heads_far_apart(lens):
    """Heads more than 2^24 bytes apart: the bits of heads that lie side by side, in chunks and row by row."""
    import ray_ops
    rays = ray_set(lens)
    n = rays[3]
    set_ = ray_ops.RaySet(*(t.cuda() for t in rays[:3]))
    x = [t.cuda() for t in inputs(n, 2, 4, 64, 64, torch.bfloat16, seed=1)]
    y = [_apart(t) for t in x]
    assert n > 140000 - 28 and y[0].stride(1) * 2 > 1 << 24 and y[2].stride(1) * 2 > 1 << 24 and y[3].stride(1) == n
    train = len(lens) < 10000
    a, b = ray_ops.ray_delta(*x, set_, marks=train), ray_ops.ray_delta(*y, set_, marks=train)
    assert torch.equal(a[0], b[0])
    if train:
        do = torch.randn(n, 4, 64, device="cuda").to(torch.bfloat16)
        ga, gb = ray_ops.ray_delta_backward(do, *x, a[2], set_), ray_ops.ray_delta_backward(_apart(do), *y, b[2], set_)
        assert all(torch.equal(p, q) for p, q in zip(ga[:5], gb[:5]))


def test_gradients_of_any_layout():
    """A gradient of o that comes head-major, with rows 2^24 bytes apart, or broadcast."""
    import ray_ops
    rays = ray_set([40, 24])
    set_ = ray_ops.RaySet(*(t.cuda() for t in rays[:3]))
    x = [t.cuda().requires_grad_() for t in inputs(rays[3], 1, 2, 16, 32, torch.bfloat16, seed=2)]
    o = ray_ops.RayDelta.apply(*x, set_)[0]
    do = torch.randn(rays[3], 2, 32, device="cuda").to(torch.bfloat16)
    want = torch.autograd.grad(o, x, do, retain_graph=True)
    far = torch.empty(rays[3], 1 << 23, dtype=torch.bfloat16, device="cuda").as_strided(do.shape, (1 << 23, 32, 1)).copy_(do)
    for g in (_apart(do), far):
        assert g.stride() != do.stride()
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(o, x, g, retain_graph=True), want))
    one = torch.autograd.grad(o, x, torch.ones_like(o), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(o.sum(), x), one))
