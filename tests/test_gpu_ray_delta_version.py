"""States that are moved on in place: a backward pass that has saved them is an error, as after any change in place."""
import pytest
import torch

from delta_oracle import inputs
from ray_oracle import ray_set

pytestmark = pytest.mark.gpu


def _make():
    import ray_ops
    rays = ray_set([3, 20])
    x = [t.cuda() for t in inputs(rays[3], 1, 1, 16, 16, torch.float32, seed=1)]
    return x, ray_ops.RaySet(*(t.cuda() for t in rays[:3])), torch.randn(2, 1, 16, 16, device="cuda")


def test_saved_states():
    import ray_ops
    x, set_, state = _make()
    leaf = [t.clone().requires_grad_() for t in x]
    o, _ = ray_ops.RayDelta.apply(*leaf, set_, state)
    want = torch.autograd.grad(o.sum(), leaf, retain_graph=True)
    ray_ops.ray_delta(*x, set_, h0=state, last=True)  # elsewhere: the saved ones are as they were
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(o.sum(), leaf, retain_graph=True), want))
    ray_ops.ray_delta(*x, set_, h0=state, last=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o.sum(), leaf)


def test_part_of_a_larger_tensor():
    """A view is written, and the tensor that it is of was saved."""
    import ray_ops
    x, set_, state = _make()
    both = torch.stack((state, state))
    w = torch.ones_like(both, requires_grad=True)
    y = (w * both).sum()
    ray_ops.ray_delta(*x, set_, h0=both[1], last=both[1])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_inference():
    import ray_ops
    x, set_, state = _make()
    want = ray_ops.ray_delta(*x, set_, h0=state, last=True)[1]
    with torch.inference_mode():
        mine = state.clone()
        assert ray_ops.ray_delta(*x, set_, h0=mine, last=mine)[1] is mine
    assert torch.equal(mine, want)
    assert ray_ops.ray_delta(*x, set_, h0=mine, last=mine)[1] is mine
