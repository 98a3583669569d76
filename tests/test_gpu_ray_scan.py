"""The gated recurrence along rays against its 64-bit oracle: forward and backward, element by element."""
import pytest
import torch

from ray_oracle import Scan, close, ray_set

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
LENS = [5, 0, 1, 15, 16, 17, 2, 0, 130, 33, 64]


def _dev_set(rays):
    import ray_ops
    return ray_ops.RaySet(*(x.cuda() for x in rays[:3]))


def _inputs(rays, C, ty, seed, shift=-2.0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    n, R = rays[3], len(rays[0])
    return ((1.5 * rnd(n, C) + shift).to(ty), rnd(n, C).to(ty), rnd(n, C).to(ty), rnd(R, C), rnd(R, C))


def _check(gate, x, dh, h0, dlast, rays, reverse, dev=None):
    import ray_ops
    ref = Scan(gate, x, rays, h0, reverse)
    c = lambda y: None if y is None else y.cuda()  # noqa: E731
    gd, xd, dd = dev or (c(gate), c(x), c(dh))
    rd = _dev_set(rays)
    h, last, marks = ray_ops.ray_scan(gd, xd, rd, h0=c(h0), reverse=reverse, marks=True)
    close(h, ref.h, ref.h_bound(x.dtype), "h")
    close(last, ref.last, 1.1 * ref.eps * ref.last_mag + 2.0 ** -126, "last")
    plain = ray_ops.ray_scan(gd, xd, rd, h0=c(h0), reverse=reverse)
    assert torch.equal(plain[0], h) and torch.equal(plain[1], last) and plain[2] is None
    got = ray_ops.ray_scan_backward(dd, gd, xd, marks, rd, dlast=c(dlast), h0=c(h0), reverse=reverse)
    for y, (want, bound), name in zip(got, ref.backward(dh, dlast, x.dtype), ("dgate", "dx", "dh0")):
        close(y, want, bound, name)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("C", [1, 3, 8, 37, 64, 130])
def test_rays_of_every_length(ty, reverse, C):
    rays = ray_set(LENS, gap=3)
    _check(*_inputs(rays, C, TYPES[ty], seed=C), rays, reverse)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
def test_no_start_and_no_gradient_of_the_end(ty, reverse):
    rays = ray_set([20, 0, 3])
    gate, x, dh, _, _ = _inputs(rays, 16, TYPES[ty], seed=1)
    _check(gate, x, dh, None, None, rays, reverse)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("lens", [[9000], [1, 5000, 0, 3000, 2]])
def test_long_sequences(ty, reverse, lens):
    rays = ray_set(lens, gap=1)
    _check(*_inputs(rays, 4, TYPES[ty], seed=2, shift=-4.0), rays, reverse)


def test_one_row_and_none():
    for lens in ([1], [0, 0], [0, 1, 0]):
        for reverse in (False, True):
            rays = ray_set(lens)
            _check(*_inputs(rays, 8, torch.float32, seed=3), rays, reverse)


@pytest.mark.parametrize("ty", TYPES)
def test_open_and_closed_gates(ty):
    """Gates of +-hundreds: z is 0 or 1 to the last bit, and nothing overflows on the way."""
    rays = ray_set([40, 3])
    gate, x, dh, h0, dlast = _inputs(rays, 8, TYPES[ty], seed=4)
    gate[::3], gate[1::3] = 300.0, -300.0
    _check(gate, x, dh, h0, dlast, rays, False)


@pytest.mark.parametrize("ty", TYPES)
def test_strides_and_alignment(ty):
    """gate and x as halves of one tensor with an odd row, gradients of a padded tensor."""
    rays = ray_set(LENS)
    for C, pad in ((16, 0), (16, 1), (6, 3)):
        gate, x, dh, h0, dlast = _inputs(rays, C, TYPES[ty], seed=5)
        both = torch.cat((gate, x, torch.zeros(rays[3], pad, dtype=x.dtype)), 1).cuda()
        wide = torch.cat((torch.zeros(rays[3], 1, dtype=x.dtype), dh), 1).cuda()
        _check(gate, x, dh, h0, dlast, rays, True, dev=(both[:, :C], both[:, C:2 * C], wide[:, 1:]))


def test_rows_of_no_ray_and_other_rays():
    """Infinities and NaN outside a ray, or in another ray, do not reach it; rows of no ray are 0."""
    import ray_ops
    rays = ray_set([20, 9, 70], gap=2)
    ids = rays[2]
    gate, x, dh, h0, dlast = _inputs(rays, 8, torch.bfloat16, seed=6)
    sick = (ids == 1) | (ids > 3)
    for y in (gate, x, dh):
        y[sick] = float("nan")
    h0[1], dlast[1] = float("inf"), float("nan")
    rd = _dev_set(rays)
    h, last, marks = ray_ops.ray_scan(gate.cuda(), x.cuda(), rd, h0=h0.cuda(), marks=True)
    got = ray_ops.ray_scan_backward(dh.cuda(), gate.cuda(), x.cuda(), marks, rd, dlast=dlast.cuda(), h0=h0.cuda())
    well, none = ~sick, ids > 3
    for y in (h, got[0], got[1]):
        assert torch.isfinite(y[well.cuda()].float()).all() and not y[none.cuda()].any()
    assert torch.isfinite(last[[0, 2]]).all() and torch.isfinite(got[2][[0, 2]]).all()


def test_offsets_past_32_bits():
    import ray_ops
    rays = ray_set([150, 150])
    gate, x, dh, h0, dlast = _inputs(rays, 8, torch.bfloat16, seed=7)
    stride = 1 << 24
    wide = torch.empty(300 * stride, dtype=torch.bfloat16, device="cuda")
    dev = []
    for i, y in enumerate((gate, x, dh)):
        w = torch.as_strided(wide, (300, 8), (stride, 1), storage_offset=i * 8)
        w.copy_(y)
        dev.append(w)
    _check(gate, x, dh, h0, dlast, rays, False, dev=tuple(dev))


@pytest.mark.parametrize("lens", [LENS, [3000, 2000]])
def test_other_stream_graph_and_repeats(lens):
    import ray_ops
    rays = ray_set(lens)
    gate, x, dh, h0, dlast = (y.cuda() for y in _inputs(rays, 16, torch.float16, seed=8))
    rd = _dev_set(rays)

    def call():
        h, last, marks = ray_ops.ray_scan(gate, x, rd, h0=h0, marks=True)
        return (h, last, *ray_ops.ray_scan_backward(dh, gate, x, marks, rd, dlast=dlast, h0=h0))

    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for _ in range(3):
        for y in held:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_in_pieces():
    """A ray's rows in two calls, the second from the first's last state, are one call (new samples chunk by chunk)."""
    import ray_ops
    rays = ray_set([40, 25])
    gate, x, _, _, _ = (y.cuda() for y in _inputs(rays, 16, torch.float32, seed=9))
    whole = ray_ops.ray_scan(gate, x, _dev_set(rays))
    head = torch.cat((torch.arange(30), torch.arange(40, 60)))
    tail = torch.cat((torch.arange(30, 40), torch.arange(60, 65)))
    a = ray_ops.ray_scan(gate[head.cuda()], x[head.cuda()], _dev_set(ray_set([30, 20])))
    b = ray_ops.ray_scan(gate[tail.cuda()], x[tail.cuda()], _dev_set(ray_set([10, 5])), h0=a[1])
    assert torch.equal(whole[0][head.cuda()], a[0]) and torch.equal(whole[0][tail.cuda()], b[0])
    assert torch.equal(whole[1], b[1])


def test_autograd_is_compositing():
    """Back to front with opacities sigmoid(gate), the last state is the composited colour; its gradients match
    differences of the compositing sum in 64 bits."""
    import ray_ops
    rays = ray_set([12, 0, 30])
    g = torch.Generator().manual_seed(10)
    gate, rgb = torch.randn(42, 1, generator=g), torch.rand(42, 3, generator=g)
    rd = _dev_set(rays)
    gd, cd = gate.cuda().requires_grad_(), rgb.cuda().requires_grad_()
    _, colour = ray_ops.RayScan.apply(gd.expand(-1, 3).contiguous(), cd, rd, None, True)
    (colour ** 2).sum().backward()

    def composite(gate, rgb):
        out = torch.zeros(3, 3, dtype=torch.float64)
        for r in range(3):
            T = 1.0
            for i in range(int(rays[1][r]), int(rays[1][r] + rays[0][r])):
                z = torch.sigmoid(gate[i])
                out[r] += T * z * rgb[i]
                T = T * (1 - z)
        return out

    want = composite(gate.double(), rgb.double())
    assert float((colour.detach().cpu().double() - want).abs().max()) < 2.0 ** -24 * 8 * 30
    f = lambda a, b: (composite(a, b) ** 2).sum()  # noqa: E731
    d = [torch.randn(y.shape, generator=g, dtype=torch.float64) for y in (gate, rgb)]
    e = 1e-6
    slope = float(f(gate + e * d[0], rgb + e * d[1]) - f(gate - e * d[0], rgb - e * d[1])) / (2 * e)
    parts = [y.grad.cpu().double() * z for y, z in zip((gd, cd), d)]
    assert abs(slope - sum(float(p.sum()) for p in parts)) < 2.0 ** -18 * sum(float(p.abs().sum()) for p in parts)


def test_python_refusals():
    import ffn_lib as fl
    import ray_ops
    rays = _dev_set(ray_set([4, 3]))
    x = torch.zeros(7, 8, device="cuda")
    with pytest.raises(fl.FfnError, match="shape"):
        ray_ops.ray_scan(x[:6], x, rays)
    with pytest.raises(fl.FfnError, match="h0 must be"):
        ray_ops.ray_scan(x, x, rays, h0=torch.zeros(2, 4, device="cuda"))
    with pytest.raises(fl.FfnError, match="last axis"):
        ray_ops.ray_scan(x.t().contiguous().t(), x, rays)
    with pytest.raises(fl.FfnError, match="marks"):
        ray_ops.ray_scan_backward(x, x, x, torch.zeros(3, device="cuda"), rays)
