"""The gated recurrence with gates far open and far closed: z and 1 - z each keep their relative accuracy."""
import pytest
import torch

from ray_oracle import F64, TINY, U, close, ray_set

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
u = 2.0 ** -24


def _with_errors(gate, x, dh, rays, h0, dlast, reverse, dtype):
    """Values and gradients in 64 bits, each with a bound that follows single precision's roundings step by step.  z and
    1 - z are off by e = (|gate| + 8) u of themselves: the rounding of gate log2(e) times its size, and a unit for each
    of exp2, sum, reciprocal and product.  A walk by parts rounds a state's share (factor, sum) separately: twice that."""
    counts, offsets, _, n = rays
    gate, x, dh = gate.to(F64), x.to(F64), dh.to(F64)
    z, keep, e = torch.sigmoid(gate), torch.sigmoid(-gate), (gate.abs() + 8) * u
    zeros = lambda: torch.zeros(n, x.shape[1], dtype=F64)  # noqa: E731
    h, eh, dx, ex, dg, eg, prev, eprev = (zeros() for _ in range(8))
    last, dh0 = h0.to(F64).clone(), dlast.to(F64).clone()
    elast, edh0 = torch.zeros_like(last), torch.zeros_like(dh0)
    for r in range(len(counts)):
        rows = list(range(int(offsets[r]), int(offsets[r]) + int(counts[r])))
        rows = rows[::-1] if reverse else rows
        s, es = last[r].clone(), elast[r].clone()
        for i in rows:
            prev[i], eprev[i] = s, es
            new = keep[i] * s + z[i] * x[i]
            es = keep[i] * es + (e[i] + u) * keep[i] * s.abs() + (e[i] + 2 * u) * z[i] * x[i].abs() + u * new.abs()
            s = new
            h[i], eh[i] = s, es
        last[r], elast[r] = s, es
        d, ed = dh0[r].clone(), edh0[r].clone()
        for i in reversed(rows):
            D = d + dh[i]
            eD = ed + u * D.abs()
            dx[i], ex[i] = z[i] * D, z[i] * eD + (e[i] + u) * (z[i] * D).abs()
            zk, far = z[i] * keep[i], (x[i] - prev[i]).abs()
            dg[i] = zk * (x[i] - prev[i]) * D
            eg[i] = zk * (far * eD + D.abs() * (eprev[i] + u * far)) + (2 * e[i] + 3 * u) * dg[i].abs()
            d, ed = keep[i] * D, keep[i] * eD + (e[i] + u) * (keep[i] * D).abs()
        dh0[r], edh0[r] = d, ed
    t = TINY[dtype]
    out = lambda y, err: (y, 2 * err + 1.1 * U[dtype] * y.abs() + t)  # noqa: E731
    state = lambda y, err: (y, 2 * err + 2.0 ** -126)  # noqa: E731
    return dict(h=out(h, eh), last=state(last, elast), dgate=out(dg, eg), dx=out(dx, ex), dh0=state(dh0, edh0))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("lens", [[5, 0, 1, 40, 17], [3000, 0, 1500]])
@pytest.mark.parametrize("lo,hi", [(-20.0, 20.0), (8.0, 20.0), (-20.0, -8.0)])
def test_far_gates(ty, reverse, lens, lo, hi):
    """Rays short enough for a walk each, and a few long ones by parts.  Every second channel's x is 0, so that what is
    left of a state is all there is."""
    import ray_ops
    rays = ray_set(lens, gap=1)
    n, R, dtype = rays[3], len(lens), TYPES[ty]
    g = torch.Generator().manual_seed(41)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    gate = (lo + (hi - lo) * torch.rand(n, 6, generator=g)).to(dtype)
    x, dh, h0, dlast = rnd(n, 6).to(dtype), rnd(n, 6).to(dtype), rnd(R, 6), rnd(R, 6)
    x[:, ::2] = 0.0
    dh[:, ::3] = 0.0
    want = _with_errors(gate, x, dh, rays, h0, dlast, reverse, dtype)
    rd = ray_ops.RaySet(*(y.cuda() for y in rays[:3]))
    gd, xd = gate.cuda(), x.cuda()
    h, last, marks = ray_ops.ray_scan(gd, xd, rd, h0=h0.cuda(), reverse=reverse, marks=True)
    dgate, dx, dh0 = ray_ops.ray_scan_backward(dh.cuda(), gd, xd, marks, rd, dlast=dlast.cuda(), h0=h0.cuda(), reverse=reverse)
    for name, y in dict(h=h, last=last, dgate=dgate, dx=dx, dh0=dh0).items():
        close(y, *want[name], name)
