"""The gated recurrence by parts of the packed rows: rays stay independent of each other."""
import functools

import pytest
import torch

from ray_oracle import Scan, close, ray_set

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
LENS = [200, 3000, 100, 2500, 40, 0, 1500]


@functools.lru_cache
def _well(ty, reverse):
    rays = ray_set(LENS, gap=2)
    g = torch.Generator().manual_seed(31)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    n, R = rays[3], len(LENS)
    inputs = ((1.5 * rnd(n, 4) - 2.0).to(TYPES[ty]), rnd(n, 4).to(TYPES[ty]), rnd(n, 4).to(TYPES[ty]), rnd(R, 4), rnd(R, 4))
    gate, x, dh, h0, dlast = inputs
    ref = Scan(gate, x, rays, h0, reverse)
    return rays, inputs, ref, ref.backward(dh, dlast, TYPES[ty])


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("sick", [0, 1, 3, 6])
@pytest.mark.parametrize("bad", ["nan", "inf", "-inf"])
def test_sick_ray(ty, reverse, sick, bad):
    """One value of a ray, and of the rows of no ray all of them, are infinite or NaN: every other ray keeps its values and
    gradients.  A NaN of the ray itself stays in it to its end, however little the gates leave of it."""
    import ray_ops
    rays, inputs, ref, bounds = _well(ty, reverse)
    counts, offsets, ids, n = rays
    gate, x, dh, h0, dlast = (y.clone() for y in inputs)
    o, c = int(offsets[sick]), int(counts[sick])
    early, late = o + c // 8, o + c - 1 - c // 8
    if reverse:
        early, late = late, early
    value = float(bad)
    none = ids >= len(LENS)
    for y in (gate, x, dh):
        y[none] = value
    x[early, 0] = value
    gate[early, 1] = float("nan")
    dh[late, 2] = value
    h0[sick, 3], dlast[sick, 3] = value, value
    rd = ray_ops.RaySet(*(y.cuda() for y in rays[:3]))
    cuda = [y.cuda() for y in (gate, x, dh, h0, dlast)]
    h, last, marks = ray_ops.ray_scan(cuda[0], cuda[1], rd, h0=cuda[3], reverse=reverse, marks=True)
    got = ray_ops.ray_scan_backward(cuda[2], cuda[0], cuda[1], marks, rd, dlast=cuda[4], h0=cuda[3], reverse=reverse)
    well = ~none & (ids != sick)
    rays_well = torch.arange(len(LENS)) != sick
    close(h[well.cuda()], ref.h[well], ref.h_bound(TYPES[ty])[well], "h")
    close(last[rays_well.cuda()], ref.last[rays_well], (1.1 * ref.eps * ref.last_mag + 2.0 ** -126)[rays_well], "last")
    for y, (want, bound), name, w in zip(got, bounds, ("dgate", "dx", "dh0"), (well, well, rays_well)):
        close(y[w.cuda()], want[w], bound[w], name)
    for y in (h, got[0], got[1]):
        assert not y[none.cuda()].any(), "rows of no ray are 0"
    # the ray's own: from the bad value on in the direction of the walk, and back from it in the gradients' direction
    after = slice(o, early + 1) if reverse else slice(early, o + c)
    before = slice(late, o + c) if reverse else slice(o, late + 1)
    finite = torch.isfinite(h.cpu().float())
    assert finite[:, 2][ids == sick].all() and not finite[after, 1].any()
    dx, last = got[1].cpu().float(), last.cpu()
    if bad == "nan":
        assert not finite[after, 0].any() and not finite[o:o + c, 3].any()
        assert not torch.isfinite(dx[before, 2]).any() and not torch.isfinite(dx[o:o + c, 3]).any()
        assert not torch.isfinite(last[sick][[0, 1, 3]]).any() and not torch.isfinite(got[2].cpu()[sick][[2, 3]]).any()
