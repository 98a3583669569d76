"""The delta rule's results as a whole, ray by ray and head by head, within a rounding of the formulas in 64 bits."""
import pytest

from delta_whole import CASES, make, off, wanted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case", CASES, ids=str)
def test_whole(case):
    import ray_ops
    rays, x, h0, do, dlast = make(case)
    want = wanted(case, rays, x, h0, do, dlast)
    set_ = ray_ops.RaySet(*(t.cuda() for t in rays[:3]))
    cx = [t.cuda() for t in x]
    opt = dict(h0=None if h0 is None else h0.cuda(), reverse=case[7])
    o, last, m = ray_ops.ray_delta(*cx, set_, last=True, marks=True, **opt)
    grads = ray_ops.ray_delta_backward(do.cuda(), *cx, m, set_, dlast=None if dlast is None else dlast.cuda(), **opt)
    got = dict(zip(("o", "last", "dq", "dk", "dv", "ddecay", "dbeta", "dh0"), (o, last, *grads)))
    assert not off(case, rays, got, want)
