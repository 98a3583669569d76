"""The delta rule on 16-bit rows rounds once, at the end: its results are those of the same values in float32, rounded."""
import pytest
import torch

from delta_oracle import inputs
from ray_oracle import ray_set

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G,dk,dv,reverse", [(2, 2, 32, 32, False), (1, 2, 64, 64, False), (2, 2, 24, 40, True), (2, 2, 16, 48, False),
                                               (2, 4, 64, 16, False), (1, 2, 40, 104, True), (1, 1, 128, 128, False)])
def test_one_rounding(H, G, dk, dv, reverse, dtype):
    """Two results in float that are 2^-22 of a row's size apart, as sums in float of some hundred terms are, fall on two sides
    of a border between neighbouring values of the type once in 2^-22 / eps of the values of that size, and more often among
    smaller ones, whose steps are finer: 8 times as often for values spread as a normal distribution is, about, twice that for
    decays' gradients, which are sums over rows.  Allowed is four times as much.  An operand held in two parts of 8 bits is off
    by 2^-16 to 2^-18 of itself, and gives 16 to 64 times as many."""
    import ray_ops
    lens = [900, 3, 0, 700, 16, 250, 1, 31, 65, 500]
    rays = ray_set(lens)
    n, R = rays[3], len(lens)
    set_ = ray_ops.RaySet(*(t.cuda() for t in rays[:3]))
    x = [t.cuda() for t in inputs(n, H, G, dk, dv, dtype, seed=dk + dv)]
    g = torch.Generator().manual_seed(7)
    h0, dlast = (torch.randn(R, G, dk, dv, generator=g).cuda() for _ in range(2))
    do = torch.randn(n, G, dv, generator=g).to(dtype).cuda()

    def both(x, do):
        o, last, m = ray_ops.ray_delta(*x, set_, h0=h0, last=True, marks=True, reverse=reverse)
        return (o, *ray_ops.ray_delta_backward(do, *x, m, set_, dlast=dlast, h0=h0, reverse=reverse)[:5])

    got, want = both(x, do), both([t.float() for t in x], do.float())
    off = {name: float((a != b.to(dtype)).float().mean())
           for name, a, b in zip(("o", "dq", "dk", "dv", "ddecay", "dbeta"), got, want)}
    most = 4 * 8 * 2.0 ** -22 / torch.finfo(dtype).eps
    assert all(v <= (2 if name == "ddecay" else 1) * most for name, v in off.items()), (most, off)
