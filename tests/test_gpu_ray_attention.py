"""Ray attention against its 64-bit oracle: forward and backward, element by element."""
import pytest
import torch

from ray_oracle import Attention, close, ray_set, seen_mask

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
LENS = [5, 0, 1, 63, 64, 65, 2, 0, 130, 17]


def _dev_set(rays):
    import ray_ops
    return ray_ops.RaySet(*(x.cuda() for x in rays[:3]))


def _inputs(qs, ks, H, G, D, ty, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda n, h: (torch.randn(n, h, D, generator=g) * spread).to(ty)  # noqa: E731
    q, k, v, do = rnd(qs[3], H), rnd(ks[3], G), rnd(ks[3], G), rnd(qs[3], H)
    return q, k, v, do, torch.rand(qs[3], generator=g) * 3, torch.rand(ks[3], generator=g) * 3


def _check(q, k, v, do, qs, ks, backward=True, *, t_q=None, t_k=None, slopes=None, scale=None, cap=0.0, causal=False,
           prefix=None, dev=None):
    """dev: device versions of q, k, v, do where they are not plain copies."""
    import ray_ops
    scale = q.shape[2] ** -0.5 if scale is None else scale
    ref = Attention(q, k, v, seen_mask(qs, ks, causal, prefix), scale=scale, cap=cap, slopes=slopes, t_q=t_q, t_k=t_k)
    c = lambda x: None if x is None else x.cuda()  # noqa: E731
    qd, kd, vd, dd = dev or (c(q), c(k), c(v), c(do))
    rq = _dev_set(qs)
    rk = rq if ks is qs else _dev_set(ks)
    opt = dict(t_q=c(t_q), t_k=c(t_k), slopes=c(slopes), scale=scale, cap=cap, causal=causal, prefix=c(prefix))
    o, lse = ray_ops.ray_attention(qd, kd, vd, rq, rk, **opt)
    close(o, ref.o, ref.o_bound(q.dtype), "o")
    close(lse, ref.lse, ref.lse_bound(), "lse")
    if backward:
        got = ray_ops.ray_attention_backward(dd, qd, kd, vd, o, lse, rq, rk, **opt)
        for x, (want, bound), name in zip(got, ref.backward(do, q.dtype), ("dq", "dk", "dv")):
            close(x, want, bound, name)
    return o, lse


OPTIONS = {
    "plain": dict(),
    "causal": dict(causal=True),
    "prefix": dict(causal=True, prefix=True),
    "cap": dict(cap=4.0),
    "bias": dict(slopes=True),
    "all": dict(causal=True, prefix=True, cap=6.0, slopes=True),
}


def _options(name, H, rays, t_q, t_k):
    o = dict(OPTIONS[name])
    if o.pop("prefix", False):
        o["prefix"] = torch.tensor([(3 * r) % 40 for r in range(rays)], dtype=torch.int32)
    if o.pop("slopes", False):
        o |= dict(slopes=torch.tensor([2.0 / (1 + h) for h in range(H)]), t_q=t_q, t_k=t_k)
    return o


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("option", OPTIONS)
def test_rays_of_every_length(ty, option):
    rays = ray_set(LENS, gap=3)
    q, k, v, do, t, _ = _inputs(rays, rays, 4, 2, 32, TYPES[ty], seed=1)
    _check(q, k, v, do, rays, rays, **_options(option, 4, len(LENS), t, t))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("D,H,G", [(8, 1, 1), (16, 3, 1), (24, 2, 2), (40, 4, 4), (64, 6, 2), (72, 2, 1), (128, 2, 2)])
def test_head_layouts(ty, D, H, G):
    rays = ray_set([70, 3, 0, 41])
    q, k, v, do, t, _ = _inputs(rays, rays, H, G, D, TYPES[ty], seed=2)
    _check(q, k, v, do, rays, rays, **_options("all", H, 4, t, t))


@pytest.mark.parametrize("ty", TYPES)
def test_one_row_and_none(ty):
    for lens in ([1], [0, 0], [0, 1, 0]):
        rays = ray_set(lens)
        q, k, v, do, _, _ = _inputs(rays, rays, 2, 1, 16, TYPES[ty], seed=3)
        _check(q, k, v, do, rays, rays)


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk", [([1, 1, 1, 1, 1], [9, 0, 1, 700, 64]), ([1, 0, 1, 1, 1], [9, 4, 1, 300, 0]),
                                   ([4, 9, 0, 3, 40], [60, 3, 5, 0, 130]), ([2, 2, 2, 2, 2], [1, 200, 2, 0, 7])])
def test_queries_of_another_set(ty, causal, nq, nk):
    """One query a ray, a ray's newest rows against all of them, and more queries than keys (rows that see nothing)."""
    qs, ks = ray_set(nq), ray_set(nk, gap=5)
    q, k, v, do, t_q, t_k = _inputs(qs, ks, 4, 2, 32, TYPES[ty], seed=4)
    for option in ("all" if causal else "bias", "causal" if causal else "plain"):
        _check(q, k, v, do, qs, ks, **_options(option, 4, len(nq), t_q, t_k))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("H,G,D", [(2, 2, 64), (8, 1, 24), (24, 1, 16)])
def test_few_queries_over_long_rays(ty, H, G, D):
    """Split over the keys and joined; 24 heads that share one key head take two passes of 16 columns."""
    qs, ks = ray_set([1, 1, 1]), ray_set([4096, 1, 2500])
    q, k, v, do, t_q, t_k = _inputs(qs, ks, H, G, D, TYPES[ty], seed=5)
    _check(q, k, v, do, qs, ks, backward=H == 2, **_options("bias", H, 3, t_q, t_k))
    _check(q, k, v, do, qs, ks, backward=False, causal=True)


FEW = [([2, 1, 0, 16, 3], [900, 64, 30, 1, 2049]), ([3, 2, 0, 5, 4, 2], [9, 60, 5, 33, 0, 64])]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("H,G,D", [(4, 2, 32), (6, 2, 64), (20, 1, 16), (2, 1, 128), (3, 3, 24)])
@pytest.mark.parametrize("nq,nk", FEW)
def test_few_queries_a_ray(ty, H, G, D, nq, nk):
    """A query at a time, split over long rays' keys and not, forward and backward."""
    qs, ks = ray_set(nq, gap=2), ray_set(nk, gap=3)
    q, k, v, do, t_q, t_k = _inputs(qs, ks, H, G, D, TYPES[ty], seed=16)
    for option in ("bias", "all"):
        _check(q, k, v, do, qs, ks, **_options(option, H, len(nq), t_q, t_k))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("nq,nk", FEW)
def test_few_queries_beside_a_sick_ray(ty, nq, nk):
    """Keys, values and gradients of one ray that are infinite or NaN leave the others' results as they are."""
    import ray_ops
    qs, ks = ray_set(nq, gap=2), ray_set(nk, gap=3)
    q, k, v, do, _, _ = _inputs(qs, ks, 4, 2, 32, TYPES[ty], seed=17)
    rq, rk = _dev_set(qs), _dev_set(ks)
    run = []
    for sick in (False, True):
        qd, kd, vd, dd = (x.clone() for x in (q, k, v, do))
        if sick:
            for x, ids in ((kd, ks[2]), (vd, ks[2]), (dd, qs[2])):
                x[ids == 3] = torch.tensor([float("nan"), float("inf")], dtype=x.dtype)[torch.arange(int((ids == 3).sum())) % 2][:, None, None]
        qd, kd, vd, dd = (x.cuda() for x in (qd, kd, vd, dd))
        o, lse = ray_ops.ray_attention(qd, kd, vd, rq, rk)
        run.append((o, lse, *ray_ops.ray_attention_backward(dd, qd, kd, vd, o, lse, rq, rk)))
    for a, b, ids in zip(*run, (qs[2], qs[2], qs[2], ks[2], ks[2])):
        well = (ids != 3).cuda()
        assert torch.equal(a[well], b[well])


@pytest.mark.parametrize("ty", ["bf16", "fp16"])
def test_long_ray_with_its_gradients(ty):
    rays = ray_set([1000, 30])
    q, k, v, do, t, _ = _inputs(rays, rays, 2, 1, 64, TYPES[ty], seed=6)
    _check(q, k, v, do, rays, rays, **_options("prefix", 2, 2, t, t))


def test_fp16_gradients_of_any_size():
    """Upstream gradients far under and over 1 keep their relative accuracy until the result leaves the type."""
    rays = ray_set([300, 9])
    q, k, v, do, _, _ = _inputs(rays, rays, 2, 2, 32, torch.float16, seed=7)
    for by in (2.0 ** -12, 2.0 ** 8):
        _check(q, k, v, (do.float() * by).half(), rays, rays)


@pytest.mark.parametrize("ty", TYPES)
def test_large_and_equal_scores(ty):
    """Scores of +-hundreds (the softmax nearly picks one key) and all equal ones."""
    rays = ray_set([90, 5])
    q, k, v, do, _, _ = _inputs(rays, rays, 2, 2, 32, TYPES[ty], seed=8, spread=8.0)
    _check(q, k, v, do, rays, rays, scale=0.5)
    _check(torch.zeros_like(q), k, v, do, rays, rays)


@pytest.mark.parametrize("ty", TYPES)
def test_what_is_not_seen_does_not_matter(ty):
    """Rows of no ray hold infinities and NaN, and so does a whole other ray: the rest stays exact, forward and
    backward; that ray's own results are not finite."""
    rays = ray_set([20, 7, 50, 1], gap=4)
    counts, offsets, ids, n = rays
    q, k, v, do, _, _ = _inputs(rays, rays, 2, 1, 32, TYPES[ty], seed=9)
    import ray_ops
    out = ids >= 4
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")])
    sick = out | (ids == 1)
    qs, ks, vs, ds = (x.clone() for x in (q, k, v, do))
    for x in (qs, ks, vs, ds):
        x[sick] = bad[torch.arange(int(sick.sum())) % 3].to(x.dtype)[:, None, None]
    rd = _dev_set(rays)
    for causal in (False, True):
        a = [x.cuda() for x in (q, k, v)]
        b = [x.cuda() for x in (qs, ks, vs)]
        o, lse = ray_ops.ray_attention(*a, rd, causal=causal)
        o2, lse2 = ray_ops.ray_attention(*b, rd, causal=causal)
        g = ray_ops.ray_attention_backward(do.cuda(), *a, o, lse, rd, causal=causal)
        g2 = ray_ops.ray_attention_backward(ds.cuda(), *b, o2, lse2, rd, causal=causal)
        ref = Attention(q, k, v, seen_mask(rays, rays, causal, None), scale=32 ** -0.5)
        well = ~sick
        close(o2[well], ref.o[well], ref.o_bound(q.dtype)[well], "o")
        assert torch.equal(lse2[well], lse[well])
        for x, (want, bound), name in zip(g2, ref.backward(do, q.dtype), ("dq", "dk", "dv")):
            close(x[well], want[well], bound[well], name)
        for x in (o2, *g2):
            assert not x[out.cuda()].any(), "rows of no ray are 0"
            assert not torch.isfinite(x[(ids == 1).cuda()].float()).all()
        assert (lse2[out.cuda()] == -float("inf")).all()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("D", [32, 56])
@pytest.mark.parametrize("option", ["plain", "prefix", "all"])
def test_longer_rays(ty, D, option):
    """Long rays on average, some of them short: wavefronts of 32 rows in 16 bits."""
    lens = [400, 150, 1, 0, 333]
    rays = ray_set(lens, gap=1)
    q, k, v, do, t, _ = _inputs(rays, rays, 4, 2, D, TYPES[ty], seed=18)
    _check(q, k, v, do, rays, rays, **_options(option, 4, len(lens), t, t))


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_longer_rays_beside_a_sick_one(ty, causal):
    """As test_what_is_not_seen_does_not_matter, where wavefronts take 32 rows."""
    import ray_ops
    rays = ray_set([300, 180, 7, 250], gap=4)
    ids = rays[2]
    q, k, v, do, _, _ = _inputs(rays, rays, 2, 1, 64, TYPES[ty], seed=19)
    sick = (ids >= 4) | (ids == 1)
    bad = torch.tensor([float("nan"), float("inf"), -float("inf")])
    qs, ks, vs, ds = (x.clone() for x in (q, k, v, do))
    for x in (qs, ks, vs, ds):
        x[sick] = bad[torch.arange(int(sick.sum())) % 3].to(x.dtype)[:, None, None]
    rd = _dev_set(rays)
    a = [x.cuda() for x in (qs, ks, vs)]
    o, lse = ray_ops.ray_attention(*a, rd, causal=causal)
    got = ray_ops.ray_attention_backward(ds.cuda(), *a, o, lse, rd, causal=causal)
    ref = Attention(q, k, v, seen_mask(rays, rays, causal, None), scale=64 ** -0.5)
    well = ~sick
    close(o[well], ref.o[well], ref.o_bound(q.dtype)[well], "o")
    close(lse[well], ref.lse[well], ref.lse_bound()[well], "lse")
    for x, (want, bound), name in zip(got, ref.backward(do, q.dtype), ("dq", "dk", "dv")):
        close(x[well], want[well], bound[well], name)


@pytest.mark.parametrize("ty", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 56])
@pytest.mark.parametrize("option,sick", [("plain", False), ("all", False), ("causal", True)])
def test_longer_rays_of_many_heads(ty, D, option, sick):
    """Enough heads for wavefronts of 32 rows; the first and the last heads are looked at."""
    import ray_ops
    lens, H, G = [400, 150, 1, 0, 349], 224, 112
    rays = ray_set(lens, gap=1)
    ids = rays[2]
    q, k, v, do, t, _ = _inputs(rays, rays, H, G, D, TYPES[ty], seed=20)
    opt = _options(option, H, len(lens), t, t)
    given = [x.clone() for x in (q, k, v, do)]
    well = torch.ones(rays[3], dtype=torch.bool)
    if sick:
        well = ids != 1
        for x in given:
            x[~well] = torch.tensor([float("nan"), float("inf")], dtype=x.dtype)[torch.arange(int((~well).sum())) % 2][:, None, None]
    qd, kd, vd, dd = (x.cuda() for x in given)
    on = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in opt.items()}
    rd = _dev_set(rays)
    o, lse = ray_ops.ray_attention(qd, kd, vd, rd, **on)
    got = ray_ops.ray_attention_backward(dd, qd, kd, vd, o, lse, rd, **on)
    for h in (0, H - 2):
        hs, gs = slice(h, h + 2), slice(h // 2, h // 2 + 1)
        some = dict(opt)
        if "slopes" in some:
            some["slopes"] = some["slopes"][hs]
        mask = seen_mask(rays, rays, some.pop("causal", False), some.pop("prefix", None))
        ref = Attention(q[:, hs], k[:, gs], v[:, gs], mask, scale=D ** -0.5, **some)
        close(o[:, hs][well], ref.o[well], ref.o_bound(q.dtype)[well], "o")
        close(lse[:, hs][well], ref.lse[well], ref.lse_bound()[well], "lse")
        for x, at, (want, bound), name in zip(got, (hs, gs, gs), ref.backward(do[:, hs], q.dtype), ("dq", "dk", "dv")):
            close(x[:, at][well], want[well], bound[well], name)


def test_infinite_value_that_is_seen():
    rays = ray_set([6, 40])
    q, k, v, do, _, _ = _inputs(rays, rays, 1, 1, 16, torch.bfloat16, seed=10)
    v[3, 0, 5] = float("inf")
    import ray_ops
    o, _ = ray_ops.ray_attention(q.cuda(), k.cuda(), v.cuda(), _dev_set(rays))
    assert (o[:6, 0, 5] == float("inf")).all() and torch.isfinite(o[6:]).all() and torch.isfinite(o[:6, 0, :5]).all()


@pytest.mark.parametrize("ty", ["bf16", "fp32"])
def test_strides(ty):
    """q, k, v as parts of one packed tensor, a head-major tensor, depths as a column of the march's samples."""
    import ray_ops
    rays = ray_set(LENS)
    n = rays[3]
    q, k, v, do, t, _ = _inputs(rays, rays, 4, 4, 24, TYPES[ty], seed=11)
    packed = torch.stack((q, k, v), 1).cuda()
    by_head = do.transpose(0, 1).contiguous().cuda().transpose(0, 1)
    dev = (packed[:, 0], packed[:, 1], packed[:, 2], by_head)
    opt = _options("all", 4, len(LENS), t, t)
    _check(q, k, v, do, rays, rays, dev=dev, **opt)
    samples = torch.rand(n, 4)
    samples[:, 3] = t
    column = samples.cuda()[:, 3]
    rd = _dev_set(rays)
    a = [x.cuda() for x in (q, k, v)]
    kw = dict(slopes=opt["slopes"].cuda(), causal=True)
    one = ray_ops.ray_attention(*a, rd, t_q=column, t_k=column, **kw)
    two = ray_ops.ray_attention(*a, rd, t_q=t.cuda(), t_k=t.cuda(), **kw)
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


def test_offsets_past_32_bits():
    """Rows whose element offsets pass 2^31: a cache with a wide row stride."""
    import ray_ops
    rays = ray_set([200, 100])
    q, k, v, do, _, _ = _inputs(rays, rays, 2, 2, 32, torch.bfloat16, seed=12)
    stride = 1 << 24  # 300 rows: 5 * 2^30 elements
    wide = torch.empty(300 * stride, dtype=torch.bfloat16, device="cuda")
    views = []
    for i, x in enumerate((q, k, v, do)):
        w = torch.as_strided(wide, (300, 2, 32), (stride, 32, 1), storage_offset=i * 64)
        w.copy_(x)
        views.append(w)
    _check(q, k, v, do, rays, rays, dev=tuple(views), causal=True)
    one = ray_set([1, 1])
    q1 = q[:2].contiguous()
    o, _ = ray_ops.ray_attention(q1.cuda(), views[1], views[2], _dev_set(one), _dev_set(rays))
    ref = Attention(q1, k, v, seen_mask(one, rays, False, None), scale=32 ** -0.5)
    close(o, ref.o, ref.o_bound(q.dtype), "o")


def test_other_stream_graph_and_repeats():
    """The same bits on another stream, in every replay of a graph, and in every call."""
    import ray_ops
    rays = ray_set(LENS)
    one = ray_set([1] * len(LENS))
    q, k, v, do, t, _ = _inputs(rays, rays, 2, 1, 32, torch.bfloat16, seed=13)
    q, k, v, do = (x.cuda() for x in (q, k, v, do))
    rd, od = _dev_set(rays), _dev_set(one)
    q1 = q[:len(LENS)].contiguous()

    def call():
        o, lse = ray_ops.ray_attention(q, k, v, rd, causal=True)
        return (o, lse, *ray_ops.ray_attention_backward(do, q, k, v, o, lse, rd, causal=True),
                *ray_ops.ray_attention(q1, k, v, od, rd))

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
        for x in held:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held))


def test_autograd_and_directional_difference():
    """RayAttention's gradients, and the slope of its values along a random direction (single precision)."""
    import ray_ops
    rays = ray_set([40, 0, 3])
    q, k, v, do, t, _ = _inputs(rays, rays, 2, 1, 16, torch.float32, seed=14)
    rd = _dev_set(rays)
    opt = dict(causal=True, cap=5.0)
    x = [y.cuda().requires_grad_() for y in (q, k, v)]
    (ray_ops.RayAttention.apply(*x, rd, None, opt) * do.cuda()).sum().backward()
    seen = seen_mask(rays, rays, True, None)
    f = lambda *y: (Attention(*y, seen, scale=0.25, cap=5.0).o * do.double()).sum()  # noqa: E731
    g = torch.Generator().manual_seed(15)
    d = [torch.randn(y.shape, generator=g, dtype=torch.float64) for y in (q, k, v)]
    e = 1e-6
    up, down = ([y.double() + s * e * z for y, z in zip((q, k, v), d)] for s in (1, -1))
    slope = float(f(*up) - f(*down)) / (2 * e)
    mine = sum(float((y.grad.cpu().double() * z).sum()) for y, z in zip(x, d))
    size = sum(float((y.grad.cpu().double() * z).abs().sum()) for y, z in zip(x, d))
    assert abs(slope - mine) < 2.0 ** -18 * size


def test_python_refusals():
    import ffn_lib as fl
    import ray_ops
    rays = _dev_set(ray_set([4, 3]))
    x = torch.zeros(7, 2, 16, device="cuda")
    with pytest.raises(fl.FfnError, match="shape"):
        ray_ops.ray_attention(x[:6], x, x, rays)
    with pytest.raises(fl.FfnError, match="must be torch.float32"):
        ray_ops.ray_attention(x, x.half(), x, rays)
    with pytest.raises(fl.FfnError, match="not float32"):
        ray_ops.ray_attention(x.double(), x.double(), x.double(), rays)
    with pytest.raises(fl.FfnError, match="need t_q"):
        ray_ops.ray_attention(x, x, x, rays, slopes=torch.ones(2, device="cuda"))
    with pytest.raises(fl.FfnError, match="prefixes"):
        ray_ops.ray_attention(x, x, x, rays, prefix=torch.zeros(5, dtype=torch.int32, device="cuda"))
    with pytest.raises(fl.FfnError, match="last axis"):
        ray_ops.ray_attention(x.transpose(1, 2).contiguous().transpose(1, 2), x, x, rays)
    with pytest.raises(fl.FfnError, match="is on cpu"):
        ray_ops.ray_attention(x.cpu(), x, x, rays)
