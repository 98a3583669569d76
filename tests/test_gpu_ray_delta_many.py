"""The delta rule for many rays, whose kernels take other turns and loads than those for few: a ray's results are the bits
that it has in a call of its own size."""
import pytest
import torch

from delta_oracle import inputs
from ray_oracle import ray_set

pytestmark = pytest.mark.gpu


def _part(rays, lo, hi):
    """Rays lo .. hi - 1 of a set without gaps, and their rows."""
    import ray_ops
    counts, offsets, ids, _ = rays
    a = int(offsets[lo])
    b = int(offsets[hi - 1] + counts[hi - 1])
    return ray_ops.RaySet(counts[lo:hi].cuda(), (offsets[lo:hi] - a).cuda(), (ids[a:b] - lo).cuda()), slice(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G,dk,dv,reverse", [(4, 4, 32, 32, False), (2, 4, 16, 40, True), (1, 2, 64, 64, False), (4, 4, 24, 16, True),
                                               (1, 1, 128, 24, False)])
def test_many_rays(H, G, dk, dv, reverse, dtype):
    import ray_ops
    R = 4400 // G
    g = torch.Generator().manual_seed(G + dk)
    lens = torch.empty(R).exponential_(1 / 12, generator=g).long()
    lens[::5] = 0
    lens[torch.randperm(R, generator=g)[:12]] = torch.tensor([33, 64, 65, 90, 100, 128, 129, 17, 80, 70, 96, 75])
    rays = ray_set(lens.tolist())
    n = rays[3]
    x = [t.cuda() for t in inputs(n, H, G, dk, dv, dtype, seed=1)]
    h0 = torch.randn(R, G, dk, dv, device="cuda")
    do, dlast = torch.randn(n, G, dv, device="cuda").to(dtype), torch.randn(R, G, dk, dv, device="cuda")

    def run(set_, rows, rays_):
        y = [t[rows] for t in x]
        o, last, m = ray_ops.ray_delta(*y, set_, h0=h0[rays_], last=True, marks=True, reverse=reverse)
        return o, last, ray_ops.ray_delta_backward(do[rows], *y, m, set_, dlast=dlast[rays_], h0=h0[rays_], reverse=reverse)

    whole = run(*_part(rays, 0, R), slice(0, R))
    step = max(1, 200 // G)
    for lo in range(0, R, max(step, R // 4)):
        hi = min(R, lo + step)
        set_, rows = _part(rays, lo, hi)
        o, last, grads = run(set_, rows, slice(lo, hi))
        assert torch.equal(o, whole[0][rows]) and torch.equal(last, whole[1][lo:hi])
        for a, b in zip(grads[:5], whole[2][:5]):
            assert torch.equal(a, b[rows])
        assert torch.equal(grads[5], whole[2][5][lo:hi])


def test_more_blocks_than_an_axis_counts():
    """More than 2^23 rays, nearly all of them empty: the last ones are not forgotten."""
    import ray_ops
    R = (1 << 23) + 77
    counts, offsets = torch.zeros(R, dtype=torch.int32), torch.zeros(R, dtype=torch.int32)
    held = [3, 1 << 22, (1 << 23) - 1, 1 << 23, R - 1]
    ids = torch.empty(20 * len(held), dtype=torch.int32)
    for i, r in enumerate(held):
        counts[r], offsets[r] = 20, 20 * i
        ids[20 * i:20 * i + 20] = r
    x = [t.cuda() for t in inputs(100, 1, 1, 8, 8, torch.float32, seed=1)]
    do = torch.randn(100, 1, 8, device="cuda")
    few = ray_ops.RaySet(*(t.cuda() for t in ray_set([20] * 5)[:3]))
    many = ray_ops.RaySet(counts.cuda(), offsets.cuda(), ids.cuda())
    res = []
    for s in (few, many):
        o, _, m = ray_ops.ray_delta(*x, s, marks=True)
        res.append((o, *ray_ops.ray_delta_backward(do, *x, m, s)[:5]))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    # and row by row
    want = ray_ops.ray_delta(*x, few)[0]
    got = ray_ops.ray_delta(*x, many)[0]
    assert float((want - got).abs().max()) < 2.0 ** -18 * float(want.abs().max())


def test_rows_of_no_ray_and_no_rays():
    """Rows that no ray holds give 0 in every output, also where there is no ray at all."""
    import ray_ops
    for H, G in ((2, 2), (1, 2)):
        x = [t.cuda() for t in inputs(2100, H, G, 16, 16, torch.bfloat16, seed=1)]
        i = torch.zeros(0, dtype=torch.int32, device="cuda")
        ids = torch.full((2100,), 5, dtype=torch.int32, device="cuda")
        s = ray_ops.RaySet(i, i, ids)
        o, last, m = ray_ops.ray_delta(*x, s, last=True, marks=True)
        grads = ray_ops.ray_delta_backward(torch.randn_like(o), *x, m, s)
        assert not o.any() and last.shape[0] == 0 and all(not t.any() for t in grads[:5])


def test_rows_past_32_bit_offsets():
    """More than 2^32 bytes between the first row and the last: the bits of rows that lie together."""
    import ray_ops
    n, apart = 600, 1 << 22
    rays = ray_set([300, 17, 283])
    x = [t.cuda() for t in inputs(n, 1, 1, 32, 32, torch.bfloat16, seed=2)]
    do = torch.randn(n, 1, 32, device="cuda").to(torch.bfloat16)
    big = torch.empty(n, apart, dtype=torch.bfloat16, device="cuda")
    far = []
    for i, t in enumerate((*x[:3], do)):
        v = big.as_strided((n, 1, 32), (apart, 32, 1), 64 * i)
        v.copy_(t)
        far.append(v)
    set_ = ray_ops.RaySet(*(t.cuda() for t in rays[:3]))
    a, b = ray_ops.ray_delta(*x, set_, marks=True), ray_ops.ray_delta(*far[:3], *x[3:], set_, marks=True)
    assert torch.equal(a[0], b[0])
    ga = ray_ops.ray_delta_backward(do, *x, a[2], set_)
    gb = ray_ops.ray_delta_backward(far[3], *far[:3], *x[3:], b[2], set_)
    assert all(torch.equal(p, q) for p, q in zip(ga[:5], gb[:5]))
