"""Layer norm and its gradients against the formula in 64 bits.

Bounds: u = eps / 2 of a type is half a step.  The row's statistics are sums of at most 16384 values in float, taken by
lanes that hold 32 at most and then by halves, so that each is off by less than 48 float steps of the sum of its terms'
sizes; y = d rstd w + b then has four roundings more, and one to the type.  The mean that is taken off is so off by up to
48 u mean|x - mean|, and mean|x - mean| rstd <= sqrt(var) rstd <= 1: xhat is off by 48 u in absolute terms, beside what is
relative to it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def formula(x, w, b, eps, dy=None):
    x = x.detach().cpu().double().requires_grad_()
    w = (torch.ones(x.shape[1]) if w is None else w.detach().cpu()).double().requires_grad_()
    b = (torch.zeros(x.shape[1]) if b is None else b.detach().cpu()).double().requires_grad_()
    mean = x.mean(1)
    rstd = 1 / torch.sqrt(((x - mean[:, None]) ** 2).mean(1) + eps)
    y = (x - mean[:, None]) * rstd[:, None] * w + b
    if dy is None:
        return y.detach(), mean.detach(), rstd.detach()
    return torch.autograd.grad(y, (x, w, b), dy.cpu().double())


def make(n, width, dtype, seed=0, shift=0.5):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, width, generator=g) + shift).to(dtype).cuda()
    w = (1 + 0.3 * torch.randn(width, generator=g)).cuda()
    b = (0.2 * torch.randn(width, generator=g)).cuda()
    dy = torch.randn(n, width, generator=g).to(dtype).cuda()
    return x, w, b, dy


def off(a, b):
    return (a.detach().cpu().double() - b).abs()


def check(x, w, b, dy, eps=1e-5):
    import ray_ops
    u = torch.finfo(x.dtype).eps / 2
    y, mean, rstd = ray_ops.layer_norm(x, w, b, eps=eps)
    ey, em, er = formula(x, w, b, eps)
    size = x.cpu().double().abs().mean(1)
    assert (off(mean, em) <= 50 * U32 * size + 1e-30).all()
    assert (off(rstd, er) <= 100 * U32 * er).all()
    wd, bd = (0 if t is None else t.cpu().double().abs() for t in (w, b))
    wd = 1.0 if w is None else wd
    xhat = (x.cpu().double() - em[:, None]).abs() * er[:, None]
    assert (off(y, ey) <= u * ey.abs() + 110 * U32 * (xhat * wd + bd) + 48 * U32 * wd
            + torch.finfo(x.dtype).smallest_normal).all()
    dx, dw, db = ray_ops.layer_norm_backward(dy, x, w, mean, rstd)
    ex, ew, eb = formula(x, w, b, eps, dy)
    g = dy.cpu().double() * wd
    # dx = rstd (g - mean(g) - xhat mean(g xhat)): each term to its own size
    terms = er[:, None] * (g.abs() + g.abs().mean(1, keepdim=True) + xhat * (g.abs() * xhat).mean(1, keepdim=True))
    assert (off(dx, ex) <= u * ex.abs() + 320 * U32 * terms + torch.finfo(x.dtype).smallest_normal).all()
    # sums over rows: float partial sums of n terms at most, each term with the roundings of xhat
    n = x.shape[0]
    d = dy.cpu().double().abs()
    assert (off(dw, ew) <= (min(n, 512) + 128) * U32 * (d * xhat).sum(0) + 48 * U32 * d.sum(0) + 1e-30).all()
    assert (off(db, eb) <= (min(n, 512) + 32) * U32 * d.sum(0) + 1e-30).all()
    return y, mean, rstd, dx, dw, db


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 7, 8, 24, 64, 65, 200, 256, 333, 512, 1000, 1024, 1032, 2048, 2056, 4096, 5000, 8192, 16384])
def test_widths(width, dtype):
    check(*make(19, width, dtype, seed=width))


@pytest.mark.parametrize("n", [1, 2, 3, 31, 4097, 70001])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows(n, dtype):
    check(*make(n, 40, dtype, seed=n))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    """Rows inside wider ones, rows that start anywhere, one row for all (stride 0), backwards gradients' rows."""
    x, w, b, dy = make(50, 64, dtype)
    import ray_ops
    want = check(x, w, b, dy)
    for shift, pad in ((0, 16), (3, 5), (8, 8)):
        wide = torch.full((50, 64 + pad + shift), float("nan"), dtype=dtype, device="cuda")
        wide[:, shift:shift + 64] = x
        got = check(wide[:, shift:shift + 64], w, b, dy)
        assert all(torch.allclose(p.float(), q.float(), rtol=1e-2, atol=1e-5) for p, q in zip(got, want))
    one = x[:1].expand(50, 64)
    y = ray_ops.layer_norm(one, w, b)[0]
    assert torch.equal(y, y[:1].expand(50, 64))
    dyw = torch.full((50, 80), float("nan"), dtype=dtype, device="cuda")
    dyw[:, 1:65] = dy
    check(x, w, b, dyw[:, 1:65])


@pytest.mark.parametrize("which", ["none", "weight", "bias", "typed"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parameters(which, dtype):
    x, w, b, dy = make(33, 72, dtype)
    if which == "typed":
        w, b = w.to(dtype), b.to(dtype)
    check(x, None if which in ("none", "bias") else w, None if which in ("none", "weight") else b, dy)


@pytest.mark.parametrize("shift", [1e3, -3e4])
def test_large_mean(shift):
    """Rows whose mean is far larger than their spread: the differences are exact, so the spread keeps its accuracy."""
    import ray_ops
    x, w, b, dy = make(40, 300, torch.float32, shift=shift)
    y, mean, rstd = ray_ops.layer_norm(x, w, b)
    ey, em, er = formula(x, w, b, 1e-5)
    assert (off(rstd, er) <= 64 * U32 * er).all()
    assert (off(y, ey) <= 64 * U32 * (1 + ey.abs())).all()
    dx = ray_ops.layer_norm_backward(dy, x, w, mean, rstd)[0]
    ex = formula(x, w, b, 1e-5, dy)[0]
    assert (off(dx, ex) <= 320 * U32 * (4 + ex.abs())).all()


def test_constant_rows():
    """No spread at all: xhat is 0, y is the bias, and rstd is 1 / sqrt(eps)."""
    import ray_ops
    x = torch.tensor([3.0, -1e4, 0.0, 0.1], device="cuda")[:, None].expand(4, 37).contiguous()
    w, b = torch.rand(37, device="cuda"), torch.rand(37, device="cuda")
    y, mean, rstd = ray_ops.layer_norm(x, w, b, eps=1e-3)
    assert torch.equal(y, b.expand(4, 37)) and torch.equal(mean, x[:, 0])
    assert float((rstd - 1e-3 ** -0.5).abs().max()) < 1e-4


def test_no_rows():
    import ray_ops
    x, w = torch.empty(0, 48, device="cuda"), torch.ones(48, device="cuda")
    y, mean, rstd = ray_ops.layer_norm(x, w)
    dx, dw, db = ray_ops.layer_norm_backward(x, x, w, mean, rstd)
    assert y.shape == dx.shape == (0, 48) and not dw.any() and not db.any()


@pytest.mark.parametrize("width", [40, 333, 3000])
def test_sick_rows_stay_alone(width):
    """A row with a NaN or an infinity gives NaN in that row; the others' bits are those without it."""
    import ray_ops
    x, w, b, dy = make(21, width, torch.bfloat16)
    y, mean, rstd = ray_ops.layer_norm(x, w, b)
    dx = ray_ops.layer_norm_backward(dy, x, w, mean, rstd)[0]
    sick = x.clone()
    sick[4, 3], sick[17, width - 1] = float("nan"), float("inf")
    y2, mean2, rstd2 = ray_ops.layer_norm(sick, w, b)
    dx2 = ray_ops.layer_norm_backward(dy, sick, w, mean2, rstd2)[0]
    ok = torch.ones(21, dtype=torch.bool, device="cuda")
    ok[4] = ok[17] = False
    assert torch.equal(y[ok], y2[ok]) and torch.equal(dx[ok], dx2[ok])
    assert y2[~ok].isnan().all() and dx2[~ok].isnan().all()


def test_needs_and_repeat():
    """Only what is asked for; the same bits again."""
    import ray_ops
    x, w, b, dy = make(9000, 64, torch.bfloat16)
    y, mean, rstd = ray_ops.layer_norm(x, w, b)
    dx, dw, db = ray_ops.layer_norm_backward(dy, x, w, mean, rstd)
    again = ray_ops.layer_norm_backward(dy, x, w, mean, rstd)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1]) and torch.equal(db, again[2])
    a = ray_ops.layer_norm_backward(dy, x, w, mean, rstd, need_dw=False)
    assert torch.equal(a[0], dx) and a[1] is None and a[2] is None
    a = ray_ops.layer_norm_backward(dy, x, w, mean, rstd, need_dx=False)
    assert a[0] is None and torch.equal(a[1], dw) and torch.equal(a[2], db)


def test_autograd():
    import ray_ops
    x, w, b, dy = make(77, 40, torch.float32)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    ray_ops.LayerNorm.apply(x, w, b, 1e-4).backward(dy)
    for t, e in zip((x, w, b), formula(x, w, b, 1e-4, dy)):
        assert float(off(t.grad, e).max()) < 1e-5 * max(1.0, float(e.abs().max()))
    y = ray_ops.LayerNorm.apply(x, w, b)
    g, = torch.autograd.grad((y ** 2).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        g.sum().backward()


def test_gradient_against_differences():
    """The gradient of a scalar of y against central differences of the 64-bit formula, of x and of the parameters."""
    import ray_ops
    x, w, b, dy = make(6, 24, torch.float32, seed=3)
    y, mean, rstd = ray_ops.layer_norm(x, w, b)
    grads = ray_ops.layer_norm_backward(dy, x, w, mean, rstd)
    args = [t.cpu().double() for t in (x, w, b)]
    f = lambda x, w, b: float((formula(x, w, b, 1e-5)[0] * dy.cpu().double()).sum())  # noqa: E731
    g = torch.Generator().manual_seed(1)
    for i in range(3):
        d = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-5 * d, args[i] - 1e-5 * d
        num = (f(*up) - f(*down)) / 2e-5
        assert abs(num - float((grads[i].cpu().double() * d).sum())) < 1e-4 * (1 + abs(num))


def test_graph_and_stream():
    """Captured and replayed with new inputs, and on a stream of its own: the eager bits."""
    import ray_ops
    x, w, b, dy = make(5000, 64, torch.bfloat16)

    def both(x, dy):
        y, mean, rstd = ray_ops.layer_norm(x, w, b)
        return (y, mean, rstd) + ray_ops.layer_norm_backward(dy, x, w, mean, rstd)

    sx, sdy = x.clone(), dy.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        on_stream = both(sx, sdy)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(on_stream, both(x, dy)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(sx, sdy)
    for seed in (5, 6, 7):
        x2, _, _, dy2 = make(5000, 64, torch.bfloat16, seed=seed)
        sx.copy_(x2)
        sdy.copy_(dy2)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, both(x2, dy2)))


def test_rows_past_32_bit_offsets():
    """More than 2^32 bytes between the first row and the last."""
    import ray_ops
    n, width, apart = 70, 64, 1 << 26
    big = torch.empty(n, apart // 2, dtype=torch.bfloat16, device="cuda")
    x, w, b, dy = make(n, width, torch.bfloat16)
    far = big[:, :width]
    far.copy_(x)
    y, mean, rstd = ray_ops.layer_norm(far, w, b)
    assert torch.equal(y, ray_ops.layer_norm(x, w, b)[0])
    assert torch.equal(ray_ops.layer_norm_backward(dy, far, w, mean, rstd)[0],
                       ray_ops.layer_norm_backward(dy, x, w, mean, rstd)[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("typed", [False, True])
def test_parameters_anywhere(typed, dtype):
    """Parameters that do not start on 16 bytes: the bits of those that do."""
    import ray_ops
    x, w, b, dy = make(30, 256, dtype)
    if typed:
        w, b = w.to(dtype), b.to(dtype)
    wide = torch.zeros(2, 260, dtype=w.dtype, device="cuda")
    wide[0, 1:257], wide[1, 3:259] = w, b
    p, q = wide[0, 1:257], wide[1, 3:259]
    y, mean, rstd = ray_ops.layer_norm(x, w, b)
    assert torch.equal(y, ray_ops.layer_norm(x, p, q)[0])
    for s, t in zip(ray_ops.layer_norm_backward(dy, x, w, mean, rstd), ray_ops.layer_norm_backward(dy, x, p, mean, rstd)):
        assert torch.equal(s, t)
