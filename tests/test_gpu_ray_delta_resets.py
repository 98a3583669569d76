"""Decays' gradients where nothing passes a row: 0, and no trace of the sums that cancel there."""
import pytest
import torch

from delta_oracle import inputs
from ray_oracle import ray_set

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G,dk,dv", [(1, 2, 32, 32), (1, 1, 64, 64), (2, 2, 16, 40), (1, 1, 128, 16)])
@pytest.mark.parametrize("reverse", [False, True])
def test_gradients_of_resets(H, G, dk, dv, reverse, dtype):
    import ray_ops
    lens = [50, 1, 0, 37, 16]
    rays = ray_set(lens)
    n = rays[3]
    set_ = ray_ops.RaySet(*(t.cuda() for t in rays[:3]))
    x = inputs(n, H, G, dk, dv, dtype, seed=4)
    places = [0, 3, 15, 16, 17, 31, 32, 40, 49]
    x[3][places, 0] = -float("inf")
    x[3][[51 + p for p in (5, 20)]] = -1000.0  # past the first ray and that of one row: exp gives 0 as well
    cx = [t.cuda() for t in x]
    g = torch.Generator().manual_seed(1)
    h0, dlast = (torch.randn(len(lens), G, dk, dv, generator=g).cuda() for _ in range(2))
    do = torch.randn(n, G, dv, generator=g).to(dtype).cuda()
    none = torch.zeros(n, G, dtype=torch.bool)
    none[places, 0] = True
    none[[51 + p for p in (5, 20)]] = True
    for start in (True, False):
        opt = dict(h0=h0 if start else None, reverse=reverse)
        m = ray_ops.ray_delta(*cx, set_, marks=True, **opt)[2]
        dd = ray_ops.ray_delta_backward(do, *cx, m, set_, dlast=dlast, **opt)[3].cpu()
        zero = none.clone()
        if not start:
            for o, c in zip(rays[1].tolist(), lens):
                if c:
                    zero[o + c - 1 if reverse else o] = True
        assert not dd[zero].any()
        assert bool((dd[~zero] != 0).all())
