"""The delta rule along rays: values, states and gradients against the recurrence in 64 bits."""
import pytest
import torch

from delta_oracle import Delta, inputs
from ray_oracle import close, ray_set

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _cuda(rays):
    import ray_ops
    return ray_ops.RaySet(*(x.cuda() for x in rays[:3]))


def check(rays, H, G, dk, dv, dtype, seed=0, start=False, reverse=False, scale=None, keys="random", change=None):
    import ray_ops
    n, R = rays[3], len(rays[0])
    x = inputs(n, H, G, dk, dv, dtype, seed, keys)
    if change:
        change(x)
    g = torch.Generator().manual_seed(seed + 100)
    state = (R, G, dk, dv)
    h0 = torch.randn(state, generator=g) if start else None
    do, dlast = torch.randn(n, G, dv, generator=g).to(dtype), torch.randn(state, generator=g) if start else None
    # what a row of no ray holds must not matter
    outside = (rays[2] >= R)
    for t in (*x, do):
        t[outside] = float("nan")
    set_ = _cuda(rays)
    cx = [t.cuda() for t in x]
    opt = dict(h0=None if h0 is None else h0.cuda(), reverse=reverse, scale=scale)
    want = Delta(*(torch.where(outside.view(-1, *[1] * (t.dim() - 1)), 0.0, t) for t in x), rays, h0, scale, reverse)
    wo, wl = want.bounds(dtype)
    for marks in (False, True):
        o, last, m = ray_ops.ray_delta(*cx, set_, last=True, marks=marks, **opt)
        close(o, want.o, wo, "o")
        close(last, want.last, wl, "last")
    got = ray_ops.ray_delta_backward(do.cuda(), *cx, m, set_, dlast=None if dlast is None else dlast.cuda(), **opt)
    ref = want.backward(torch.where(outside.view(-1, 1, 1), 0.0, do), dlast, dtype)
    for name, t, (e, b) in zip(("dq", "dk", "dv", "ddecay", "dbeta", "dh0"), got, ref):
        if t is not None:
            close(t, e, b, name)
    again = ray_ops.ray_delta_backward(do.cuda(), *cx, m, set_, dlast=None if dlast is None else dlast.cuda(), **opt)
    assert all(p is None or torch.equal(p, q) for p, q in zip(got, again))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [[1], [2, 1, 3], [15, 16, 17], [31, 32, 33], [63, 64, 65, 1], [0, 5, 0, 0, 40, 0], [200, 3]])
def test_lengths(lens, dtype):
    check(ray_set(lens), 2, 2, 32, 32, dtype, seed=len(lens))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dk,dv", [(8, 8), (8, 128), (16, 24), (24, 40), (32, 16), (40, 8), (64, 64), (64, 16), (72, 104),
                                   (128, 8), (128, 32), (128, 128)])
def test_dims(dk, dv, dtype):
    check(ray_set([37, 5]), 1, 1, dk, dv, dtype, seed=dk + dv, start=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,G", [(1, 1), (1, 4), (3, 3), (2, 6)])
@pytest.mark.parametrize("reverse", [False, True])
def test_heads(H, G, reverse, dtype):
    check(ray_set([20, 0, 35, 1], gap=2), H, G, 16, 24, dtype, seed=H + G, start=True, reverse=reverse)


@pytest.mark.parametrize("reverse", [False, True])
def test_options(reverse):
    check(ray_set([50, 18], gap=1), 2, 2, 32, 48, torch.float32, reverse=reverse, scale=-0.7)
    check(ray_set([50, 18]), 2, 2, 32, 48, torch.float32, reverse=reverse, scale=0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alike_keys(dtype):
    """Neighbouring keys that are nearly the same, written with all their strength."""
    check(ray_set([130, 40]), 2, 2, 32, 32, dtype, keys="alike", start=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("decay", [0.0, -30.0, -200.0, -float("inf")])
def test_decays(decay, dtype):
    """No decay, decays that leave next to nothing, and resets: among the others, and for every row."""
    def some(x):
        x[3][::5] = decay

    def every(x):
        x[3][:] = decay

    def after(x):  # strong ones first: the weak ones after them keep their accuracy
        x[3][:7] = decay

    for change in (some, every, after):
        check(ray_set([45, 16]), 1, 2, 16, 16, dtype, start=True, change=change)


@pytest.mark.parametrize("beta", [0.0, 1.0, 2.0])
def test_strengths(beta):
    def change(x):
        x[4][::2] = beta

    check(ray_set([45, 16]), 1, 2, 16, 16, torch.float32, start=True, change=change)


def test_long_ray():
    check(ray_set([1500, 700]), 1, 1, 64, 64, torch.float32, start=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_next_samples(dtype):
    """Row by row from state to state, in place: what one call over all rows gives; rays that get no row keep their state."""
    import ray_ops
    R, G, dk, dv, T = 7, 2, 24, 40, 5
    x = inputs(R * T, G, G, dk, dv, dtype, seed=3)
    whole = ray_set([T] * R)
    g = torch.Generator().manual_seed(1)
    h0 = torch.randn(R, G, dk, dv, generator=g)
    want = Delta(*x, whole, h0)
    wo, wl = want.bounds(dtype)
    state = h0.cuda()
    o = torch.zeros(R * T, G, dv, dtype=dtype)
    for t in range(T):
        rows = torch.arange(R) * T + t
        one = ray_set([1] * R)
        y, last, marks = ray_ops.ray_delta(*(t_[rows].cuda() for t_ in x), _cuda(one), h0=state, last=state)
        assert last is state and marks is None
        o[rows] = y.cpu()
    close(o, want.o, wo, "o")
    close(state, want.last, wl, "last")
    keep = state.clone()
    none = _cuda((torch.zeros(R, dtype=torch.int32), torch.zeros(R, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)))
    ray_ops.ray_delta(*(t_[:0].cuda() for t_ in x), none, h0=state, last=state)
    assert torch.equal(state, keep)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("what", ["q", "k", "v", "decay", "beta"])
@pytest.mark.parametrize("at", [0, 5, 15, 16, 21, 40])
def test_sick_rows(what, at, dtype):
    """A NaN or an infinity reaches the o of its own row and of later ones of its ray at most: the rows before it and the
    other rays have the bits they have without it."""
    import ray_ops
    rays = ray_set([48, 30, 48])
    x = [t.cuda() for t in inputs(rays[3], 2, 2, 32, 40, dtype, seed=9)]
    set_ = _cuda(rays)
    o = ray_ops.ray_delta(*x, set_)[0]
    sick = [t.clone() for t in x]
    row = 78 + at
    s = sick[["q", "k", "v", "decay", "beta"].index(what)]
    s[row].view(-1)[1 if s[row].numel() > 1 else 0] = float("nan")
    s[min(row + 3, 125)].view(-1)[-1] = float("inf")
    o2 = ray_ops.ray_delta(*sick, set_)[0]
    assert torch.equal(o[:row], o2[:row])
    assert o2[row].isnan().any()
    if what == "v":  # other columns of the state hold none of it
        fine = torch.ones_like(o2, dtype=torch.bool)
        fine[row:, 0, 1] = fine[row:, 1, -1] = False
        assert torch.equal(o[fine], o2[fine])


def test_sick_rays_in_the_backward():
    """What one ray holds does not reach another's gradients."""
    import ray_ops
    rays = ray_set([20, 30, 25])
    x = [t.cuda() for t in inputs(rays[3], 2, 4, 32, 32, torch.bfloat16, seed=9)]
    do = torch.randn(rays[3], 4, 32).to(torch.bfloat16).cuda()
    set_ = _cuda(rays)

    def grads(x, do):
        m = ray_ops.ray_delta(*x, set_, marks=True)[2]
        return ray_ops.ray_delta_backward(do, *x, m, set_)[:5]

    a = grads(x, do)
    sick, sdo = [t.clone() for t in x], do.clone()
    for t in (*sick, sdo):
        t[25] = float("nan")
    sdo[30] = float("inf")
    b = grads(sick, sdo)
    ok = torch.ones(rays[3], dtype=torch.bool, device="cuda")
    ok[20:50] = False
    for p, q in zip(a, b):
        assert torch.equal(p[ok], q[ok])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    """Heads cut from one projection, and rows inside wider ones: the bits of contiguous inputs."""
    import ray_ops
    rays = ray_set([33, 20])
    x = [t.cuda() for t in inputs(rays[3], 2, 2, 32, 32, dtype, seed=5)]
    do = torch.randn(rays[3], 2, 32).to(dtype).cuda()
    set_ = _cuda(rays)
    wide = torch.full((rays[3], 4, 2, 40), float("nan"), dtype=dtype, device="cuda")
    gates = torch.full((rays[3], 5, 3), float("nan"), dtype=dtype, device="cuda")
    for i, t in enumerate((*x[:3], do)):
        wide[:, i, :, :32] = t
    gates[:, 1:3, 0], gates[:, 3:5, 2] = x[3], x[4]
    y = [wide[:, i, :, :32] for i in range(3)] + [gates[:, 1:3, 0], gates[:, 3:5, 2]]
    a, b = ray_ops.ray_delta(*x, set_, marks=True), ray_ops.ray_delta(*y, set_, marks=True)
    assert torch.equal(a[0], b[0])
    ga = ray_ops.ray_delta_backward(do, *x, a[2], set_)
    gb = ray_ops.ray_delta_backward(wide[:, 3, :, :32], *y, b[2], set_)
    assert all(torch.equal(p, q) for p, q in zip(ga[:5], gb[:5]))


def test_autograd():
    import ray_ops
    rays = ray_set([20, 0, 7])
    x = [t.cuda().requires_grad_() for t in inputs(rays[3], 1, 2, 16, 24, torch.float32, seed=5)]
    h0 = torch.randn(3, 2, 16, 24, device="cuda", requires_grad=True)
    set_ = _cuda(rays)
    o, last = ray_ops.RayDelta.apply(*x, set_, h0)
    do, dlast = torch.randn_like(o), torch.randn_like(last)
    got = torch.autograd.grad((o, last), x + [h0], (do, dlast))
    want = Delta(*(t.detach().cpu() for t in x), rays, h0.detach().cpu())
    for name, t, (e, b) in zip(("dq", "dk", "dv", "ddecay", "dbeta", "dh0"), got,
                               want.backward(do.cpu(), dlast.cpu(), torch.float32)):
        close(t, e, b, name)
    o, last = ray_ops.RayDelta.apply(*x, set_, None, dict(last=False, reverse=True))
    assert last is None
    got = torch.autograd.grad(o, x, do)
    want = Delta(*(t.detach().cpu() for t in x), rays, reverse=True)
    for name, t, (e, b) in zip(("dq", "dk", "dv", "ddecay", "dbeta"), got, want.backward(do.cpu(), None, torch.float32)):
        close(t, e, b, name)
    for t in x:
        y = ray_ops.RayDelta.apply(*x, set_)[0]
        g, = torch.autograd.grad((y ** 2).sum(), [t], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad((g ** 2).sum(), [t])


def test_graph_and_stream():
    """Captured and replayed with other rows, lengths and states; and on a stream of its own."""
    import ray_ops
    dt = torch.bfloat16

    def make(seed):
        lens = [[40, 3, 0, 17], [10, 10, 30, 10], [0, 0, 59, 1]][seed % 3]
        rays = ray_set(lens)
        g = torch.Generator().manual_seed(seed)
        return [t.cuda() for t in (*rays[:3], *inputs(60, 1, 2, 32, 32, dt, seed), torch.randn(4, 2, 32, 32, generator=g),
                                   torch.randn(60, 2, 32, generator=g).to(dt))]

    def both(c, o, i, q, k, v, g, b, h0, do):
        rays = ray_ops.RaySet(c, o, i)
        y, last, m = ray_ops.ray_delta(q, k, v, g, b, rays, h0=h0, last=True, marks=True)
        return (y, last, *ray_ops.ray_delta_backward(do, q, k, v, g, b, m, rays, h0=h0))

    held = make(0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = both(*held)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(out, both(*held)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*held)
    for seed in (1, 2, 3):
        new = make(seed)
        for h, t in zip(held, new):
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, both(*new)))
