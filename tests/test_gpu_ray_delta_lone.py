"""The delta rule where most rays have few rows, or none, and some have many: those go in chunks."""
import pytest
import torch

from delta_oracle import Delta, inputs
from ray_oracle import close, ray_set

pytestmark = pytest.mark.gpu


def _rows(lens, r):
    a = sum(lens[:r])
    return slice(a, a + lens[r])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype,H,G,dk,dv,reverse", [(torch.bfloat16, 2, 2, 32, 32, False), (torch.float32, 1, 2, 64, 48, True),
                                                     (torch.float16, 1, 1, 128, 128, False), (torch.bfloat16, 1, 1, 16, 8, True)])
def test_long_among_few(dtype, H, G, dk, dv, reverse, in_place):
    """Rays of more than eight rows have the bits that they have alone, where they are taken in chunks; all of them are right."""
    import ray_ops
    lens = [1, 9, 0, 300, 8, 2] + [0, 1, 3] * 40 + [17, 33] + [0] * 60
    rays = ray_set(lens)
    n, R = rays[3], len(lens)
    assert n <= 4 * R
    x = inputs(n, H, G, dk, dv, dtype, seed=5)
    h0 = torch.randn(R, G, dk, dv, generator=torch.Generator().manual_seed(1))
    cx, set_ = [t.cuda() for t in x], ray_ops.RaySet(*(t.cuda() for t in rays[:3]))
    state = h0.cuda()
    o, last, _ = ray_ops.ray_delta(*cx, set_, h0=state, last=state if in_place else True, reverse=reverse)
    want = Delta(*x, rays, h0, reverse=reverse)
    wo, wl = want.bounds(dtype)
    close(o, want.o, wo, "o")
    close(last, want.last, wl, "last")
    for r in (r for r in range(R) if lens[r] > 8):
        rows = _rows(lens, r)
        one = ray_ops.RaySet(*(t.cuda() for t in ray_set([lens[r]])[:3]))
        o1, last1, _ = ray_ops.ray_delta(*(t[rows] for t in cx), one, h0=h0[r:r + 1].cuda(), last=True, reverse=reverse)
        assert torch.equal(o[rows], o1) and torch.equal(last[r], last1[0]), r


def test_time_of_a_lone_ray():
    """One ray of 4096 rows among 2047 without any takes what it takes alone, and not a chain of 4096 rows (18 times that)."""
    import ray_ops
    x = [t.cuda() for t in inputs(4096, 4, 4, 64, 64, torch.bfloat16, seed=5)]
    counts = torch.zeros(2048, dtype=torch.int32)
    counts[77] = 4096
    ids = torch.full((4096,), 77, dtype=torch.int32)
    sets = [ray_ops.RaySet(counts.cuda(), torch.zeros_like(counts).cuda(), ids.cuda()),
            ray_ops.RaySet(*(t.cuda() for t in ray_set([4096])[:3]))]
    times = []
    for set_ in sets:
        best = 1e9
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            ray_ops.ray_delta(*x, set_)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        times.append(best)
    assert times[0] < 4 * times[1], times


def test_no_rays_of_many_rows():
    """Sets of up to eight rows, of one row a ray, and of rows of no ray: nothing is left undone."""
    import ray_ops
    for lens, gap in (([8], 0), ([1] * 700, 0), ([0, 2, 0], 3), ([9], 0), ([0, 0, 9, 0], 1)):
        rays = ray_set(lens, gap=gap)
        x = inputs(rays[3], 1, 1, 8, 8, torch.float32, seed=2)
        set_ = ray_ops.RaySet(*(t.cuda() for t in rays[:3]))
        o, last, _ = ray_ops.ray_delta(*(t.cuda() for t in x), set_, last=True)
        want = Delta(*x, rays)
        wo, wl = want.bounds(torch.float32)
        close(o, want.o, wo, "o")
        close(last, want.last, wl, "last")
