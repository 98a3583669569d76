"""What a query does not see changes nothing: infinities and NaN in another ray and in rows of no ray, with every option,
in every form of the kernels."""
import pytest
import torch

from ray_oracle import Attention, close, ray_set, seen_mask

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BAD = torch.tensor([float("nan"), float("inf"), -float("inf")])
OPTIONS = {
    "plain": dict(),
    "cap": dict(cap=4.0),
    "bias": dict(slopes=True),
    "causal cap": dict(causal=True, cap=4.0),
    "all": dict(causal=True, prefix=True, cap=6.0, slopes=True),
}


def _options(name, H, rays, t_q, t_k):
    o = dict(OPTIONS[name])
    if o.pop("prefix", False):
        o["prefix"] = torch.tensor([(3 * r) % 40 for r in range(rays)], dtype=torch.int32)
    if o.pop("slopes", False):
        o |= dict(slopes=torch.tensor([2.0 / (1 + h) for h in range(H)]), t_q=t_q, t_k=t_k)
    return o


def _sick(x, rows):
    """x with every value of these rows infinite or NaN, by turns."""
    x = x.clone()
    shape = (-1,) + (1,) * (x.dim() - 1)
    x[rows] = BAD[torch.arange(int(rows.sum())) % 3].to(x.dtype).view(shape)
    return x


def _check(qs, ks, H, G, D, ty, option, heads, seed):
    """Ray 1 and the rows of no ray are sick: q, k, v, the upstream gradient and the depths.  Every other row is compared
    with the oracle of well inputs, for the query heads from each of `heads` to the next key head; rows of no ray are 0
    in all of them."""
    import ray_ops
    g = torch.Generator().manual_seed(seed)
    rnd = lambda n, h: torch.randn(n, h, D, generator=g).to(TYPES[ty])  # noqa: E731
    q, k, v, do = rnd(qs[3], H), rnd(ks[3], G), rnd(ks[3], G), rnd(qs[3], H)
    t_q = torch.rand(qs[3], generator=g) * 3
    t_k = t_q if qs is ks else torch.rand(ks[3], generator=g) * 3
    R = len(qs[0])
    sq, sk = ((s[2] == 1) | (s[2] >= R) for s in (qs, ks))
    opt = _options(option, H, R, t_q, t_k)
    on = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in opt.items()}
    if "slopes" in on:
        on["t_q"], on["t_k"] = _sick(t_q, sq).cuda(), _sick(t_k, sk).cuda()
    qd, kd, vd, dd = (_sick(x, s).cuda() for x, s in ((q, sq), (k, sk), (v, sk), (do, sq)))
    rq = ray_ops.RaySet(*(x.cuda() for x in qs[:3]))
    rk = rq if qs is ks else ray_ops.RaySet(*(x.cuda() for x in ks[:3]))
    o, lse = ray_ops.ray_attention(qd, kd, vd, rq, rk, **on)
    got = ray_ops.ray_attention_backward(dd, qd, kd, vd, o, lse, rq, rk, **on)
    share = H // G
    seen = seen_mask(qs, ks, opt.get("causal", False), opt.get("prefix"))
    for kh in heads:
        hs, gs = slice(kh * share, (kh + 1) * share), slice(kh, kh + 1)
        some = {n: opt[n] for n in ("cap", "slopes", "t_q", "t_k") if n in opt}
        if "slopes" in some:
            some["slopes"] = some["slopes"][hs]
        ref = Attention(q[:, hs], k[:, gs], v[:, gs], seen, scale=D ** -0.5, **some)
        wq, wk = ~sq, ~sk
        close(o[:, hs][wq], ref.o[wq], ref.o_bound(q.dtype)[wq], "o")
        close(lse[:, hs][wq], ref.lse[wq], ref.lse_bound()[wq], "lse")
        for x, at, w, (want, bound), name in zip(got, (hs, gs, gs), (wq, wk, wk), ref.backward(do[:, hs], q.dtype),
                                                 ("dq", "dk", "dv")):
            close(x[:, at][w], want[w], bound[w], name)
    nq, nk = (qs[2] >= R).cuda(), (ks[2] >= R).cuda()
    for x, rows in zip((o, *got), (nq, nq, nk, nk)):
        assert not x[rows].any(), "rows of no ray are 0"
    assert (lse[nq] == -float("inf")).all()


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("option", OPTIONS)
@pytest.mark.parametrize("D", [32, 64, 128])
def test_sick_ray(ty, option, D):
    rays = ray_set([20, 7, 50, 0, 1], gap=4)
    _check(rays, rays, 4, 2, D, ty, option, (0, 1), seed=21)


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("option", OPTIONS)
@pytest.mark.parametrize("nq,nk", [([2, 3, 0, 16, 1], [900, 200, 30, 2049, 64]), ([1, 1, 1, 1, 1], [70, 300, 0, 1, 128])])
def test_sick_ray_few_queries(ty, option, nq, nk):
    _check(ray_set(nq, gap=2), ray_set(nk, gap=3), 4, 2, 32, ty, option, (0, 1), seed=22)


@pytest.mark.parametrize("ty", ["bf16", "fp16"])
@pytest.mark.parametrize("option", OPTIONS)
@pytest.mark.parametrize("D", [32, 56])
def test_sick_ray_two_sets_of_rows(ty, option, D):
    """Rays of 128 rows and more on average, and blocks of 128 rows for all CUs: wavefronts of 32 rows."""
    rays = ray_set([400, 150, 1, 0, 349], gap=2)
    _check(rays, rays, 224, 112, D, ty, option, (0, 55, 111), seed=23)
