"""Expert layers: the grouping exactly, products and gradients against 64 bits."""
import pytest
import torch

from ray_oracle import TINY, U, close

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def _ids(n, E, seed, none=0.1):
    """Skewed ids, an expert without rows, and rows of no expert (negative and too large ids)."""
    g = torch.Generator().manual_seed(seed)
    ids = (torch.rand(n, generator=g) ** 2 * E).long()
    if E > 2:
        ids[ids == E // 2] = 0
    out = torch.rand(n, generator=g) < none
    ids[out] = torch.where(torch.rand(int(out.sum()), generator=g) < 0.5, -1, E + 3)
    return ids.to(torch.int32)


@pytest.mark.parametrize("n,E", [(0, 3), (1, 1), (5, 1), (63, 2), (64, 64), (1000, 8), (4096, 5), (4097, 33),
                                 (100003, 7), (50000, 1024), (8192, 1024), (8193, 3)])
def test_plan(n, E):
    import ray_ops
    ids = _ids(n, E, seed=n + E)
    p = ray_ops.expert_plan(ids.cuda(), E)
    b = torch.where((ids < 0) | (ids >= E), E, ids.long())
    counts = torch.bincount(b, minlength=E + 1)
    assert torch.equal(p.counts.cpu().long(), counts[:E])
    assert torch.equal(p.offsets.cpu().long(), (torch.cumsum(counts, 0) - counts)[:E])
    assert torch.equal(p.rows.cpu().long(), torch.sort(b, stable=True)[1])


def _check(n, E, K, M, ty, seed, relu, bias=True, none=0.1):
    import ray_ops
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    ids = _ids(n, E, seed, none)
    x, W, b, dy = rnd(n, K).to(ty), (rnd(E, M, K) * K ** -0.5).to(ty), (rnd(E, M) * 0.3).to(ty), rnd(n, M).to(ty)
    # what rows of no expert hold does not matter
    out = (ids < 0) | (ids >= E)
    x[out], dy[out] = float("nan"), float("inf")
    plan = ray_ops.expert_plan(ids.cuda(), E)
    y = ray_ops.expert_linear(x.cuda(), W.cuda(), b.cuda() if bias else None, plan, relu=relu)
    u, f = U[ty], 2.0 ** -24
    want, mag = torch.zeros(n, M, dtype=torch.float64), torch.zeros(n, M, dtype=torch.float64)
    X, WW, B = x.double(), W.double(), b.double() if bias else torch.zeros(E, M, dtype=torch.float64)
    for e in range(E):
        r = ids == e
        want[r] = X[r] @ WW[e].T + B[e]
        mag[r] = X[r].abs() @ WW[e].abs().T + B[e].abs()
    if relu:
        want = want.clamp(min=0)
    close(y, want, 1.1 * (u * want.abs() + f * (K + 8) * mag) + TINY[ty], "y")
    dx, dW, db = ray_ops.expert_linear_backward(dy.cuda(), x.cuda(), W.cuda(), plan, y=y if relu else None)
    d = dy.double()
    if relu:
        d = torch.where(y.cpu().double() > 0, d, 0.0)
    gx, mx = torch.zeros(n, K, dtype=torch.float64), torch.zeros(n, K, dtype=torch.float64)
    gW, gb = torch.zeros(E, M, K, dtype=torch.float64), torch.zeros(E, M, dtype=torch.float64)
    mW, mb = torch.zeros_like(gW), torch.zeros_like(gb)
    for e in range(E):
        r = ids == e
        gx[r], mx[r] = d[r] @ WW[e], d[r].abs() @ WW[e].abs()
        gW[e], mW[e] = d[r].T @ X[r], d[r].abs().T @ X[r].abs()
        gb[e], mb[e] = d[r].sum(0), d[r].abs().sum(0)
    close(dx, gx, 1.1 * (u * gx.abs() + f * (M + 8) * mx) + TINY[ty], "dx")
    # sums of up to n products in single precision: their roundings add up as a walk, here ten of its steps
    steps = 10 * max(n, 1) ** 0.5 + 16
    close(dW, gW, 1.1 * f * steps * mW + 2.0 ** -126, "dW")
    close(db, gb, 1.1 * f * steps * mb + 2.0 ** -126, "db")


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("n,E,K,M", [(1, 1, 8, 8), (130, 3, 32, 64), (777, 9, 24, 40), (1500, 4, 136, 72),
                                     (3000, 70, 64, 64), (257, 2, 256, 8), (300, 1, 8, 256),
                                     (150, 2, 1024, 24), (150, 2, 16, 1024), (90, 1, 520, 512)])
def test_layers(ty, relu, n, E, K, M):
    _check(n, E, K, M, TYPES[ty], seed=n + K, relu=relu)


@pytest.mark.parametrize("ty", TYPES)
def test_empty_and_unassigned(ty):
    _check(0, 3, 16, 16, TYPES[ty], seed=1, relu=True)
    _check(90, 2, 16, 16, TYPES[ty], seed=2, relu=True, none=1.0)
    _check(90, 2, 16, 16, TYPES[ty], seed=3, relu=False, bias=False)


def test_long_group():
    """One expert with many chunks of rows, the others with few."""
    _check(60001, 3, 64, 32, torch.bfloat16, seed=4, relu=True)


@pytest.mark.parametrize("ty", ["bf16", "fp16"])
@pytest.mark.parametrize("n,E,K,M", [(140001, 3, 72, 136), (140001, 2, 200, 40), (90001, 3, 24, 264)])
def test_many_rows(ty, n, E, K, M):
    """Enough rows for the widest tiles of every product."""
    _check(n, E, K, M, TYPES[ty], seed=6, relu=True)


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
@pytest.mark.parametrize("K,M", [(40, 136), (136, 104)])
def test_many_experts(ty, K, M):
    """About two rows an expert, many with none."""
    _check(2500, 1020, K, M, TYPES[ty], seed=7, relu=True)


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
def test_slot_order_and_strides(ty):
    """Two layers in slot order between are the layers in row order; x as columns of a wider tensor."""
    import ray_ops
    g = torch.Generator().manual_seed(5)
    n, E, t = 700, 6, TYPES[ty]
    rnd = lambda *s: torch.randn(*s, generator=g).to(t).cuda()  # noqa: E731
    ids = _ids(n, E, 5)
    wide, W1, W2, b1, dy = rnd(n, 96), rnd(E, 32, 64) * 0.1, rnd(E, 16, 32) * 0.1, rnd(E, 32), rnd(n, 16)
    x = wide[:, 32:]
    plan = ray_ops.expert_plan(ids.cuda(), E)
    h = ray_ops.expert_linear(x, W1, b1, plan, relu=True)
    y = ray_ops.expert_linear(h, W2, None, plan)
    hs = ray_ops.expert_linear(x, W1, b1, plan, relu=True, y_slots=True)
    ys = ray_ops.expert_linear(hs, W2, None, plan, x_slots=True)
    assert torch.equal(hs, h[plan.rows.long()]) and torch.equal(ys, y)
    a = ray_ops.expert_linear_backward(dy, h, W2, plan)
    s = ray_ops.expert_linear_backward(dy, hs, W2, plan, x_slots=True)
    assert torch.equal(s[0], a[0][plan.rows.long()]) and torch.equal(s[1], a[1]) and torch.equal(s[2], a[2])
    a1 = ray_ops.expert_linear_backward(a[0], x, W1, plan, y=h)
    s1 = ray_ops.expert_linear_backward(s[0], x, W1, plan, y=hs, y_slots=True)
    assert all(torch.equal(p, q) for p, q in zip(a1, s1))


def test_nan_and_infinity_stay_in_their_rows():
    import ray_ops
    n, E = 200, 3
    g = torch.Generator().manual_seed(6)
    ids = torch.randint(0, E, (n,), generator=g, dtype=torch.int32)
    x, W = torch.randn(n, 16, generator=g).bfloat16(), torch.randn(E, 8, 16, generator=g).bfloat16()
    x[50], x[51] = float("nan"), float("inf")
    plan = ray_ops.expert_plan(ids.cuda(), E)
    y = ray_ops.expert_linear(x.cuda(), W.cuda(), None, plan, relu=True).float().cpu()
    assert torch.isnan(y[50]).all()
    rest = torch.ones(n, dtype=torch.bool)
    rest[50:52] = False
    assert torch.isfinite(y[rest]).all()


def test_offsets_past_32_bits():
    import ray_ops
    n, stride = 300, 1 << 24
    g = torch.Generator().manual_seed(7)
    x, W = torch.randn(n, 16, generator=g).bfloat16(), torch.randn(2, 8, 16, generator=g).bfloat16()
    wide = torch.empty(n * stride, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(wide, (n, 16), (stride, 1))
    far.copy_(x)
    plan = ray_ops.expert_plan(torch.arange(n, dtype=torch.int32).cuda() % 2, 2)
    dy = torch.randn(n, 8, generator=g).bfloat16().cuda()
    near = x.cuda()
    assert torch.equal(ray_ops.expert_linear(far, W.cuda(), None, plan), ray_ops.expert_linear(near, W.cuda(), None, plan))
    a, b = (ray_ops.expert_linear_backward(dy, z, W.cuda(), plan) for z in (far, near))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_other_stream_graph_and_repeats():
    import ray_ops
    n, E = 5000, 11
    g = torch.Generator().manual_seed(8)
    ids = _ids(n, E, 8).cuda()
    x, W, b, dy = (torch.randn(*s, generator=g).half().cuda() for s in ((n, 32), (E, 64, 32), (E, 64), (n, 64)))

    def call():
        plan = ray_ops.expert_plan(ids, E)
        y = ray_ops.expert_linear(x, W, b, plan, relu=True)
        return (y, plan.rows, *ray_ops.expert_linear_backward(dy, x, W, plan, y=y))

    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for _ in range(3):
        for y in held:
            y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, held))


def test_autograd():
    import ray_ops
    n, E = 120, 3
    g = torch.Generator().manual_seed(9)
    ids = torch.randint(0, E, (n,), generator=g)
    x, W, b, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((n, 16), (E, 8, 16), (E, 8), (n, 8)))
    p = [y.float().cuda().requires_grad_() for y in (x, W, b)]
    plan = ray_ops.expert_plan(ids.to(torch.int32).cuda(), E)
    (ray_ops.ExpertLinear.apply(*p, plan, True) * dy.float().cuda()).sum().backward()
    q = [y.float().double().requires_grad_() for y in (x, W, b)]
    pre = torch.einsum("nk,nmk->nm", q[0], q[1][ids]) + q[2][ids]
    (torch.relu(pre) * dy.float().double()).sum().backward()
    assert float(pre.abs().min()) > 1e-5  # no value so near 0 that single precision could decide otherwise
    for a, c in zip(p, q):
        assert float((a.grad.cpu().double() - c.grad).abs().max()) < 2.0 ** -18 * float(c.grad.abs().max()) * 4
    d = [torch.randn(y.shape, generator=g, dtype=torch.float64) for y in q]
    f = lambda x, W, b: (torch.relu(torch.einsum("nk,nmk->nm", x, W[ids]) + b[ids]) * dy.float().double()).sum()  # noqa: E731
    with torch.no_grad():
        e = 1e-8
        slope = float(f(*[y + e * z for y, z in zip(q, d)]) - f(*[y - e * z for y, z in zip(q, d)])) / (2 * e)
    parts = [a.grad.cpu().double() * z for a, z in zip(p, d)]
    assert abs(slope - sum(float(y.sum()) for y in parts)) < 1e-5 * sum(float(y.abs().sum()) for y in parts)


def test_python_refusals():
    import ffn_lib as fl
    import ray_ops
    plan = ray_ops.expert_plan(torch.zeros(5, dtype=torch.int32, device="cuda"), 2)
    x, W = torch.zeros(5, 16, device="cuda"), torch.zeros(2, 8, 16, device="cuda")
    with pytest.raises(fl.FfnError, match="shape"):
        ray_ops.expert_linear(x[:4], W, None, plan)
    with pytest.raises(fl.FfnError, match="W must be"):
        ray_ops.expert_linear(x, W[:1], None, plan)
    with pytest.raises(fl.FfnError, match="multiples of 8"):
        ray_ops.expert_linear(x[:, :12], W[:, :, :12].contiguous(), None, plan)
    with pytest.raises(fl.FfnError, match="int32"):
        ray_ops.expert_plan(torch.zeros(5, dtype=torch.int64, device="cuda"), 2)
