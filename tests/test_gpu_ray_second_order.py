"""The operators' gradients are not differentiable themselves: a second one is refused, never wrong."""
import pytest
import torch

from ray_oracle import ray_set

pytestmark = pytest.mark.gpu


def _refuses(results, inputs):
    """A penalty on the gradients beside a term that has a gradient of its own, as a loss holds them: refused for any of
    the inputs alone, and for all that the loss depends on."""
    for second in [lambda loss, x=x: torch.autograd.grad(loss, [x]) for x in inputs] + [lambda loss: loss.backward()]:
        first = torch.autograd.grad(sum((y ** 2).sum() for y in results()), inputs, create_graph=True)
        loss = sum((y ** 2).sum() for y in first) + sum((y ** 2).sum() for y in inputs)
        with pytest.raises(RuntimeError, match="differentiated once"):
            second(loss)


def _set(lens):
    import ray_ops
    return ray_ops.RaySet(*(x.cuda() for x in ray_set(lens)[:3]))


def _leaf(*shape):
    return torch.randn(*shape, device="cuda", requires_grad=True)


def test_attention():
    import ray_ops
    x = [_leaf(9, 2, 8) for _ in range(3)]
    _refuses(lambda: [ray_ops.RayAttention.apply(*x, _set([5, 4]))], x)


def test_scan():
    import ray_ops
    x = [_leaf(9, 4), _leaf(9, 4)]
    h0 = _leaf(2, 4)
    _refuses(lambda: ray_ops.RayScan.apply(*x, _set([5, 4]), h0), x + [h0])


def test_experts():
    import ray_ops
    plan = ray_ops.expert_plan(torch.tensor([0, 1, 1, 0, 2], dtype=torch.int32, device="cuda"), 3)
    x = [_leaf(5, 8), _leaf(3, 16, 8), _leaf(3, 16)]
    _refuses(lambda: [ray_ops.ExpertLinear.apply(*x, plan, True)], x)


def test_hash_encode(tmp_path):
    import numpy as np
    import ffnerf_tools as ft
    import ray_model
    spec = ft.ModelSpec(n_levels=4, f_per_level=2, log2_T=[12] * 4, res=ft.level_resolutions(4, 16.0, growth=1.5))
    nerf = ft.Nerf(str(tmp_path), "rays", spec=spec, occ=ft.OccParams(G_occ=16, box_min=np.zeros(3), box_max=np.ones(3)))
    table = torch.nn.Parameter(nerf.t["table"])
    xyz = torch.rand(50, 3, device="cuda")
    _refuses(lambda: [ray_model.HashEncode.apply(table, xyz, nerf)], [table])


def test_first_gradients_with_and_without_a_graph_are_the_same():
    import ray_ops
    x = [_leaf(9, 2, 8) for _ in range(3)]
    y = ray_ops.RayAttention.apply(*x, _set([5, 4]))
    a = torch.autograd.grad((y ** 2).sum(), x, retain_graph=True)
    b = torch.autograd.grad((y ** 2).sum(), x, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
