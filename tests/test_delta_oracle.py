"""The delta rule's oracle: its gradients against differences of its own values."""
import torch

from delta_oracle import Delta, inputs
from ray_oracle import F64, ray_set


def test_gradients_against_differences():
    rays = ray_set([5, 0, 9, 1])
    x = [t.to(F64) for t in inputs(rays[3], 2, 4, 8, 16, torch.float32, seed=1)]
    g = torch.Generator().manual_seed(2)
    h0 = torch.randn(4, 4, 8, 16, generator=g, dtype=F64)
    do, dlast = torch.randn(rays[3], 4, 16, generator=g, dtype=F64), torch.randn(4, 4, 8, 16, generator=g, dtype=F64)
    for reverse in (False, True):
        def f(args):
            d = Delta(*args[:5], rays, args[5], reverse=reverse)
            return float((d.o * do).sum() + (d.last * dlast).sum())

        args = x + [h0]
        grads = Delta(*x, rays, h0, reverse=reverse).backward(do, dlast, torch.float32)
        for i, (grad, _) in enumerate(grads):
            d = torch.randn(args[i].shape, generator=g, dtype=F64)
            up, down = list(args), list(args)
            up[i], down[i] = args[i] + 1e-6 * d, args[i] - 1e-6 * d
            num = (f(up) - f(down)) / 2e-6
            assert abs(num - float((grad * d).sum())) < 1e-6 * (1 + abs(num)), i
