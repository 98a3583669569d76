"""Tensors of one row, of one head and of none: the strides of such an axis say nothing, and are not looked at."""
import pytest
import torch

from ray_oracle import ray_set

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16]


def _strided(shape, strides, dtype):
    size = 1 + sum((n - 1) * s for n, s in zip(shape, strides)) if 0 not in shape else 1
    return torch.randn(size, device="cuda").to(dtype).as_strided(shape, strides)


def _rays(lens):
    import ray_ops
    return ray_ops.RaySet(*(x.cuda() for x in ray_set(lens)[:3]))


def _same(a, b):
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,strides,lens", [((1, 2, 16), (33, 16, 1), [0, 1]), ((5, 1, 16), (16, 3, 1), [2, 3]),
                                                ((0, 2, 16), (1, 0, 0), [0, 0]), ((1, 1, 16), (7, 5, 1), [1])])
def test_attention(dtype, shape, strides, lens):
    import ray_ops
    q, k, v, do = (_strided(shape, strides, dtype) for _ in range(4))
    rays = _rays(lens)
    plain = [x.clone(memory_format=torch.contiguous_format) for x in (q, k, v, do)]
    o, lse = ray_ops.ray_attention(q, k, v, rays)
    want = ray_ops.ray_attention(*plain[:3], rays)
    _same((o, lse), want)
    _same(ray_ops.ray_attention_backward(do, q, k, v, o, lse, rays),
          ray_ops.ray_attention_backward(plain[3], *plain[:3], *want, rays))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,strides,lens", [((1, 8), (1 << 40, 1), [0, 1]), ((0, 8), (1, 0), [0, 0])])
def test_scan(dtype, shape, strides, lens):
    import ray_ops
    gate, x, dh = (_strided(shape, strides, dtype) for _ in range(3))
    rays = _rays(lens)
    plain = [y.clone(memory_format=torch.contiguous_format) for y in (gate, x, dh)]
    h, last, marks = ray_ops.ray_scan(gate, x, rays, marks=True)
    want = ray_ops.ray_scan(*plain[:2], rays, marks=True)
    _same((h, last), want)
    _same(ray_ops.ray_scan_backward(dh, gate, x, marks, rays),
          ray_ops.ray_scan_backward(plain[2], *plain[:2], want[2], rays))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,row", [(1, 17), (1, 1 << 40), (0, 1)])
def test_experts(dtype, n, row):
    import ray_ops
    plan = ray_ops.expert_plan(torch.ones(n, dtype=torch.int32, device="cuda"), 3)
    x, dy = _strided((n, 16), (row, 1 if n else 0), dtype), _strided((n, 8), (row, 1 if n else 0), dtype)
    W = torch.randn(3, 8, 16, device="cuda").to(dtype)
    plain = [y.clone(memory_format=torch.contiguous_format) for y in (x, dy)]
    _same([ray_ops.expert_linear(x, W, None, plan)], [ray_ops.expert_linear(plain[0], W, None, plan)])
    _same(ray_ops.expert_linear_backward(dy, x, W, plan), ray_ops.expert_linear_backward(plain[1], plain[0], W, plan))
