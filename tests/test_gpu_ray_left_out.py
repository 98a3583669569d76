"""Functions of torch with their last arguments left out: the gradients that the same call has with None in their place."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _same(short, long, leaves):
    g = torch.randn_like(short)
    want = torch.autograd.grad(long, leaves, g)
    assert torch.equal(short, long)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(short, leaves, g), want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm(dtype):
    import ray_ops
    x = torch.randn(20, 48, device="cuda").to(dtype).requires_grad_()
    w, b = torch.randn(48, device="cuda", requires_grad=True), torch.randn(48, device="cuda", requires_grad=True)
    f = ray_ops.LayerNorm.apply
    _same(f(x), f(x, None, None, 1e-5), [x])
    _same(f(x, w), f(x, w, None, 1e-5), [x, w])
    _same(f(x, w, b), f(x, w, b, 1e-5), [x, w, b])
    _same(f(x.detach(), w), f(x.detach(), w, None), [w])


def test_combine():
    import ray_ops
    ids = torch.randint(-1, 4, (30, 2), dtype=torch.int32, device="cuda")
    route = ray_ops.expert_route(ids, 4)
    y = torch.randn(60, 16, device="cuda", requires_grad=True)
    _same(ray_ops.ExpertCombine.apply(y, route), ray_ops.ExpertCombine.apply(y, route, None), [y])


def test_along_rays():
    import ray_ops
    from delta_oracle import inputs
    from ray_oracle import ray_set
    rays = ray_set([9, 0, 20])
    set_ = ray_ops.RaySet(*(t.cuda() for t in rays[:3]))
    x = [t.cuda().requires_grad_() for t in inputs(rays[3], 2, 2, 16, 16, torch.float32, seed=1)]
    f = ray_ops.RayDelta.apply
    _same(f(*x, set_)[0], f(*x, set_, None, {})[0], x)
    f = ray_ops.RayAttention.apply
    _same(f(*x[:3], set_), f(*x[:3], set_, None, None), x[:3])
    gate, y = (torch.randn(rays[3], 8, device="cuda", requires_grad=True) for _ in range(2))
    f = ray_ops.RayScan.apply
    _same(f(gate, y, set_)[0], f(gate, y, set_, None, False)[0], [gate, y])
    plan = ray_ops.expert_plan(torch.randint(0, 3, (rays[3],), dtype=torch.int32, device="cuda"), 3)
    W = torch.randn(3, 8, 8, device="cuda", requires_grad=True)
    f = ray_ops.ExpertLinear.apply
    _same(f(y, W, None, plan), f(y, W, None, plan, False, False, False), [y, W])
