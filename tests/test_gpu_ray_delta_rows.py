"""The delta rule row by row (few rows a ray, no backward pass): every width that its kernels are made for, and all options."""
import pytest
import torch

from delta_oracle import Delta, inputs
from ray_oracle import close, ray_set

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
LENS = [1, 3, 0, 4, 2, 8, 0, 1, 7, 5, 0, 0]  # 31 rows of 12 rays, none of more than 8
GAPPED = [1, 3, 0, 4, 2, 8, 0, 0, 1]          # 19 rows of 9 rays, and one of no ray after each


def _cuda(rays):
    import ray_ops
    return ray_ops.RaySet(*(t.cuda() for t in rays[:3]))


def check(lens, H, G, dk, dv, dtype, reverse=False, gap=0, change=None, strided=False, scale=None, in_place=True, start=True):
    import ray_ops
    rays = ray_set(lens, gap=gap)
    n, R = rays[3], len(lens)
    assert n <= 4 * R
    x = inputs(n, H, G, dk, dv, dtype, seed=dk + dv)
    if change:
        change(x)
    h0 = torch.randn(R, G, dk, dv, generator=torch.Generator().manual_seed(dk)) if start else None
    outside = rays[2] >= R
    want = Delta(*x, rays, h0, scale, reverse)
    for t in x:
        t[outside] = float("nan")
    cx = [t.cuda() for t in x]
    if strided:  # head-major, in rows of their own width and more
        wide = [torch.full((t.shape[1], n, t.shape[2] + 8) if t.dim() == 3 else (t.shape[1], n, 3), float("nan"), dtype=dtype,
                           device="cuda") for t in cx]
        cx = [w[:, :, :t.shape[2]].transpose(0, 1).copy_(t) if t.dim() == 3 else w[:, :, 1].transpose(0, 1).copy_(t)
              for w, t in zip(wide, cx)]
        assert not any(t.is_contiguous() for t in cx if t.shape[1] > 1)
    state = None if h0 is None else h0.cuda()
    o, last, marks = ray_ops.ray_delta(*cx, _cuda(rays), h0=state, last=state if in_place and start else True, scale=scale,
                                       reverse=reverse)
    assert marks is None and (not (in_place and start) or last is state)
    wo, wl = want.bounds(dtype)
    close(o, want.o, wo, "o")
    close(last, want.last, wl, "last")
    assert not o[outside.cuda()].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk", [8, 32, 40, 64, 72, 128])
@pytest.mark.parametrize("dv", [8, 40, 64, 128])
def test_widths(dk, dv, dtype):
    check(LENS, 1, 1, dk, dv, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk,dv", [(16, 24), (64, 64), (128, 40)])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("H,G", [(1, 4), (2, 2), (2, 6)])
def test_heads_directions_gaps(H, G, reverse, dk, dv, dtype):
    check(GAPPED, H, G, dk, dv, dtype, reverse=reverse, gap=1, in_place=reverse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk,dv", [(24, 24), (64, 40), (96, 128)])
def test_strides(dk, dv, dtype):
    check(LENS, 2, 4, dk, dv, dtype, strided=True)
    check(GAPPED, 2, 2, dk, dv, dtype, strided=True, reverse=True, gap=1)


@pytest.mark.parametrize("dk", [32, 64, 128])
@pytest.mark.parametrize("decay", [0.0, -30.0, -200.0, -float("inf")])
def test_decays(decay, dk):
    def some(x):
        x[3][::3] = decay

    def every(x):
        x[3][:] = decay

    for change in (some, every):
        check(LENS, 1, 2, dk, 16, torch.float32, change=change)


def test_options():
    check(LENS, 1, 2, 64, 32, torch.float32, scale=-0.7)
    check(LENS, 1, 2, 64, 32, torch.float32, scale=0.0)
    check(LENS, 1, 2, 64, 32, torch.bfloat16, start=False)
    check([1] * 5000, 1, 1, 64, 64, torch.bfloat16)
    check([1], 1, 1, 128, 128, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dk", [32, 64, 128])
@pytest.mark.parametrize("what", ["q", "k", "v", "decay", "beta"])
def test_sick_rows(what, dk, dtype):
    """A NaN or an infinity does not reach the o of rows before it, other rays, or other heads."""
    import ray_ops
    rays = ray_set(LENS)
    x = [t.cuda() for t in inputs(rays[3], 2, 2, dk, 40, dtype, seed=9)]
    o, last, _ = ray_ops.ray_delta(*x, _cuda(rays), last=True)
    row, ray = 13, 5  # rows 10 to 17 are ray 5's
    for bad in (float("nan"), float("inf")):
        sick = [t.clone() for t in x]
        s = sick[["q", "k", "v", "decay", "beta"].index(what)]
        s[row].view(2, -1)[1, 0] = bad
        o2, last2, _ = ray_ops.ray_delta(*sick, _cuda(rays), last=True)
        fine = torch.ones_like(o, dtype=torch.bool)
        fine[row:18, 1] = False
        assert torch.equal(o[fine], o2[fine]) and not bool(torch.isfinite(o2[row, 1]).all())
        keep = torch.ones_like(last, dtype=torch.bool)
        keep[ray, 1] = False
        assert torch.equal(last[keep], last2[keep])


def test_graph_replays():
    """Captured in place, and replayed with other rows and lengths: each replay moves the states on as a call does."""
    import ray_ops
    R, dt = 6, torch.bfloat16
    sets = [ray_set(lens) for lens in ([1, 3, 0, 4, 2, 11], [2, 2, 2, 5, 10, 0], [0, 0, 20, 1, 0, 0])]
    data = [[t.cuda() for t in (*r[:3], *inputs(21, 1, 2, 64, 32, dt, seed=i))] for i, r in enumerate(sets)]
    held = [t.clone() for t in data[0]]
    start = torch.randn(R, 2, 64, 32, device="cuda")
    state = start.clone()

    def move(c, s):
        return ray_ops.ray_delta(*c[3:], ray_ops.RaySet(*c[:3]), h0=s, last=s)[0]

    move(held, state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = move(held, state)
    state.copy_(start)
    want = start.clone()
    for i in (1, 2, 0, 2):
        for h, t in zip(held, data[i]):
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        o = move(data[i], want)
        assert torch.equal(out, o) and torch.equal(state, want)
