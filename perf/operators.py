"""Operators of models that look along a ray, as cases that can be timed and checked.

`ffn_march` leaves a batch of rays as packed samples: `counts`, `offsets` per ray, `ray_ids` per sample and the samples
{x, y, z, t}.  Three operators work on that layout:

  attention   samples (or one query a ray) attend to the samples of their own ray: scaled products, an optional
              tanh cap, a bias that falls with the distance in t, a causal mask with a prefix that every sample sees
  scan        h_t = (1 - z_t) h_{t-1} + z_t x_t along each ray, z = sigmoid(gate): compositing of feature channels
  experts     each sample goes through the layer of its own expert: grouping by expert id, product, bias, ReLU

`run` in its plain form computes them by elementary torch operations in 32 bits; `exact` restates them in 64 bits.
"""
from __future__ import annotations

import math
import sys
import zlib
from pathlib import Path

import numpy as np
import torch

PKG = str(Path(__file__).resolve().parent.parent / "ffnerf-experimental_amd")
if PKG not in sys.path:
    sys.path.insert(0, PKG)

own = False
DEV = "cuda"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
STEP = math.sqrt(3.0) / 256  # the march's lattice step on the unit box


# ---------------------------------------------------------------------------
# the cases


def listed() -> list:
    return [
        # one pooled query a ray for a handful of rays: what an interactive pick asks for; launches are all of it
        dict(name="pool_few", op="attention", query="one", rays=16, mean=24, longest=64, spread="marched", heads=4,
             kv_heads=4, dim=16, type="bf16", cap=0.0, causal=False, prefix=0, train=False),
        # each ray's newest sample against its cached ones: few rows, the longest march the framework allows
        dict(name="pool_long", op="attention", query="one", rays=96, mean=0, longest=4096, spread="even", heads=8,
             kv_heads=8, dim=64, type="fp16", cap=0.0, causal=True, prefix=0, train=False),
        # a training batch of the marched step's kind: short rays of every length, every mask option
        dict(name="attend_train", op="attention", query="all", rays=8192, mean=28, longest=256, spread="marched",
             heads=4, kv_heads=4, dim=32, type="bf16", cap=20.0, causal=True, prefix=8, train=True),
        # long rays: the products rule; two query heads share a key head
        dict(name="attend_long_train", op="attention", query="all", rays=24, mean=0, longest=4096, spread="even",
             heads=4, kv_heads=2, dim=64, type="bf16", cap=0.0, causal=True, prefix=0, train=True),
        # the framework's default arithmetic, odd sizes, one key head for all
        dict(name="attend_fp32_train", op="attention", query="all", rays=3001, mean=40, longest=200,
             spread="marched", heads=3, kv_heads=1, dim=24, type="fp32", cap=15.0, causal=False, prefix=0,
             train=True),
        # a preview tile: latency counts
        dict(name="scan_small", op="scan", rays=64, mean=20, longest=64, spread="marched", channels=64, type="fp32",
             reverse=True, start=False, train=False),
        # the marched training step's batch: 2^18 rays, about 4.6 million samples
        dict(name="scan_train", op="scan", rays=262144, mean=22, longest=512, spread="marched", channels=64,
             type="bf16", reverse=False, start=False, train=True),
        # few long sequences with a state to start from: the length has to be split
        dict(name="scan_long", op="scan", rays=3, mean=0, longest=262144, spread="even", channels=128, type="fp16",
             reverse=False, start=True, train=False),
        # odd channels, the framework's default arithmetic, back to front as compositing goes
        dict(name="scan_odd_train", op="scan", rays=5003, mean=50, longest=1000, spread="marched", channels=37,
             type="fp32", reverse=True, start=True, train=True),
        # a preview's samples through the first layer of few experts, odd rows
        dict(name="experts_small", op="experts", rows=3001, experts=8, k=32, out=64, skew=1.0, type="fp32",
             relu=True, train=False),
        # a marched batch's samples through a hidden layer of a scene of many regions, some of them empty
        dict(name="experts_batch", op="experts", rows=1 << 21, experts=64, k=64, out=64, skew=1.0, type="bf16",
             relu=True, train=False),
        # the gradient of a wide layer, the largest experts with many times the rows of the smallest
        dict(name="experts_wide_train", op="experts", rows=500009, experts=24, k=256, out=256, skew=1.5, type="bf16",
             relu=True, train=True),
    ]


def _log(rng, lo, hi) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["attention", "attention", "scan", "scan", "experts", "experts"])
    ty = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "attention":
        one = rng.random() < 0.35
        longest = _log(rng, 24, 4096)
        kv = rng.choice([1, 2, 4])
        c = dict(op=op, query="one" if one else "all", rays=0, mean=0, longest=longest, spread="even",
                 heads=kv * rng.choice([1, 1, 2]), kv_heads=kv, dim=rng.choice([16, 24, 32, 64]), type=ty,
                 cap=rng.choice([0.0, 0.0, 12.5, 30.0]), causal=rng.random() < 0.6, prefix=rng.choice([0, 0, 3, 16]),
                 train=not one and rng.random() < 0.6)
        # the scores of a padded batch stay under those of the largest listed case
        most = 1.2e9 / (longest * c["heads"] * (1 if one else longest))
        c["rays"] = _log(rng, 1, int(max(1, min(most, 10000))))
        if c["rays"] >= 64 and rng.random() < 0.7:
            c["spread"], c["mean"] = "marched", max(2, longest // rng.choice([2, 4, 8]))
        return c
    if op == "scan":
        c = dict(op=op, rays=_log(rng, 1, 200000), mean=0, longest=0, spread="even",
                 channels=rng.choice([1, 3, 16, 32, 37, 64, 96, 128, 200]), type=ty, reverse=rng.random() < 0.5,
                 start=rng.random() < 0.5, train=rng.random() < 0.5)
        most = 1.2e8 / (c["channels"] * c["rays"])  # samples a ray
        c["longest"] = _log(rng, 1, int(max(1, min(most, 200000))))
        if c["rays"] >= 64 and c["longest"] >= 16 and rng.random() < 0.7:
            c["spread"], c["mean"] = "marched", max(2, c["longest"] // rng.choice([2, 5, 11]))
        return c
    k, out = rng.choice([16, 32, 64, 104, 128, 256]), rng.choice([8, 16, 64, 72, 128, 256])
    most = 1.2e8 / max(k, out)
    return dict(op=op, rows=_log(rng, 1, int(most)), experts=_log(rng, 1, 128), k=k, out=out,
                skew=rng.choice([0.0, 0.7, 1.5]), type=ty, relu=rng.random() < 0.6, train=rng.random() < 0.5)


def _fixed(c) -> np.random.RandomState:
    """Lengths and group sizes go by the case alone, so that `work` knows them."""
    return np.random.RandomState(zlib.crc32(repr(sorted((k, v) for k, v in c.items() if k != "name")).encode()))


def lengths(c) -> np.ndarray:
    """Samples a ray: marched batches have misses and many short rays, even ones fill half the march or more."""
    r, R, top = _fixed(c), c["rays"], c["longest"]
    if c["spread"] == "even":
        n = r.randint(max(1, top // 2), top + 1, R)
    else:
        n = np.minimum(r.exponential(c["mean"], R).astype(np.int64) + 1, top)
        n[r.rand(R) < 0.2] = 0
    n[r.randint(R)] = top
    return n.astype(np.int64)


def group_sizes(c) -> np.ndarray:
    """Rows an expert: sizes fall with a power of its rank; a tenth of many experts gets none."""
    r, E = _fixed(c), c["experts"]
    p = (1.0 + np.arange(E)) ** -c["skew"] * (0.5 + r.rand(E))
    if E >= 10:
        p[r.permutation(E)[:E // 10]] = 0.0
    r.shuffle(p)
    return r.multinomial(c["rows"], p / p.sum()).astype(np.int64)


def work(c) -> dict:
    b = 4 if c["type"] == "fp32" else 2
    if c["op"] == "attention":
        n, H, G, D = lengths(c).astype(np.float64), c["heads"], c["kv_heads"], c["dim"]
        N, Q = n.sum(), (n.sum() if c["query"] == "all" else len(n))
        if c["query"] == "one":
            pairs = n.sum()
        elif c["causal"]:
            pairs = (n * (n + 1) / 2).sum()
        else:
            pairs = (n * n).sum()
        bytes_ = b * D * (2 * H * Q + 2 * G * N) + 4 * H * Q + 4 * (Q + N)
        flops = 4 * D * H * pairs
        if c["train"]:  # do in, dq, dk, dv out
            bytes_ += b * D * (2 * H * Q + 2 * G * N)
            flops += 10 * D * H * pairs
        return {"bytes": float(bytes_), "flops": float(flops)}
    if c["op"] == "scan":
        N, C, R = float(lengths(c).sum()), c["channels"], c["rays"]
        units = 3 + (3 if c["train"] else 0)
        states = 1 + (1 if c["start"] else 0) + (2 if c["train"] else 0)
        return {"bytes": b * C * N * units + 4.0 * C * R * states, "flops": 8.0 * C * N * (3 if c["train"] else 1)}
    N, E, K, M = c["rows"], c["experts"], c["k"], c["out"]
    if c["train"]:  # dy, y, x, W in; dx, dW, db out
        return {"bytes": float(b * (N * (2 * M + 2 * K) + E * M * K) + 4 * E * M * (K + 1) + 4 * N),
                "flops": 4.0 * N * K * M}
    return {"bytes": float(b * (N * (K + M) + E * M * K + E * M) + 8 * N), "flops": 2.0 * N * K * M}


# ---------------------------------------------------------------------------
# inputs


def prepare(c, seed) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    ty = TYPES[c["type"]]

    def normal(*shape, dtype=ty, scale=1.0, shift=0.0):
        x = torch.empty(shape, device=DEV, dtype=torch.float32).normal_(shift, scale, generator=gen)
        return x.to(dtype)

    if c["op"] == "experts":
        N, E, K, M = c["rows"], c["experts"], c["k"], c["out"]
        sizes = group_sizes(c)
        ids = torch.repeat_interleave(torch.arange(E, device=DEV), torch.from_numpy(sizes).to(DEV))
        ids = ids[torch.randperm(N, device=DEV, generator=gen)].to(torch.int32)
        s = dict(case=c, ids=ids, most=int(sizes.max()), x=normal(N, K), W=normal(E, M, K, scale=K ** -0.5),
                 b=normal(E, M, scale=0.1))
        if c["train"]:  # the layer's output as the forward left it: half of a ReLU layer's values are 0
            s["y"] = normal(N, M).clamp_(min=0.0) if c["relu"] else normal(N, M)
            s["dy"] = normal(N, M)
        return s

    n = lengths(c)
    n = n[np.random.RandomState(int(seed) & 0x7FFFFFFF).permutation(len(n))]
    N, R = int(n.sum()), len(n)
    counts = torch.from_numpy(n).to(DEV)
    offsets = torch.cumsum(counts, 0) - counts
    ray_ids = torch.repeat_interleave(torch.arange(R, device=DEV), counts)
    place = torch.arange(N, device=DEV) - offsets[ray_ids]
    s = dict(case=c, n=N, longest=c["longest"], counts=counts.to(torch.int32), offsets=offsets.to(torch.int32),
             ray_ids=ray_ids.to(torch.int32))
    if c["op"] == "scan":
        C = c["channels"]
        s["gate"] = normal(N, C, shift=-2.0, scale=1.5)  # opacities of 0.03 to 0.4: a state lasts some ten samples
        s["x"] = normal(N, C)
        s["h0"] = normal(R, C, dtype=torch.float32) if c["start"] else None
        if c["train"]:
            s["dh"] = normal(N, C)
            s["dlast"] = normal(R, C, dtype=torch.float32)
        return s
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    samples = torch.rand(N, 4, device=DEV, generator=gen)  # {x, y, z, t}, t on the lattice of its ray
    samples[:, 3] = 0.2 + STEP * (place + 0.5)
    s["samples"] = samples
    s["k"], s["v"] = normal(N, G, D), normal(N, G, D)
    s["slopes"] = torch.tensor([2.0 ** (1 - h) for h in range(H)], device=DEV)
    s["prefix"] = torch.randint(0, c["prefix"] + 1, (R,), device=DEV, generator=gen, dtype=torch.int32) \
        if c["prefix"] else None
    if c["query"] == "all":
        s["q"] = normal(N, H, D)
    else:  # one query a ray, at the depth of its last sample
        s["q"] = normal(R, H, D)
        s["one"] = torch.ones(R, device=DEV, dtype=torch.int32)
        s["each"] = torch.arange(R, device=DEV, dtype=torch.int32)
        s["tq"] = (0.2 + STEP * (counts.to(torch.float32) - 0.5)).contiguous()
    if c["train"]:
        s["do"] = normal(N, H, D)
    return s


# ---------------------------------------------------------------------------
# one pass


def run(s):
    return {"attention": _attention, "scan": _scan, "experts": _experts}[s["case"]["op"]](s)


def _padded(counts, offsets, longest):
    """Row of each place of each ray [R, longest], and whether the place is there."""
    at = torch.arange(longest, device=counts.device)
    there = at < counts[:, None]
    return torch.where(there, offsets[:, None].long() + at, 0), there


def _attention(s):
    c = s["case"]
    scale = c["dim"] ** -0.5
    if own:
        import ray_ops
        keys = ray_ops.RaySet(s["counts"], s["offsets"], s["ray_ids"])
        queries = keys if c["query"] == "all" else ray_ops.RaySet(s["one"], s["each"], s["each"])
        tk = s["samples"][:, 3]
        opt = dict(t_q=tk if c["query"] == "all" else s["tq"], t_k=tk, slopes=s["slopes"], scale=scale, cap=c["cap"],
                   causal=c["causal"], prefix=s["prefix"])
        o, lse = ray_ops.ray_attention(s["q"], s["k"], s["v"], queries, keys, **opt)
        if not c["train"]:
            return o, lse
        return (o, lse) + tuple(ray_ops.ray_attention_backward(s["do"], s["q"], s["k"], s["v"], o, lse, queries, keys,
                                                               **opt))
    H, G = c["heads"], c["kv_heads"]
    rk, there_k = _padded(s["counts"], s["offsets"], s["longest"])
    if c["query"] == "all":
        rq, there_q, nq, tq = rk, there_k, s["counts"], s["samples"][:, 3]
    else:
        rq, there_q = _padded(s["one"], s["each"], 1)
        nq, tq = s["one"], s["tq"]

    def rays(x, rows):  # [N, heads, D] -> [R, H, L, D] in 32 bits
        return x[rows].float().permute(0, 2, 1, 3).repeat_interleave(H // x.shape[1], 1)

    q, k, v = rays(s["q"], rq), rays(s["k"], rk), rays(s["v"], rk)
    capped = torch.matmul(q, k.transpose(2, 3)) * scale
    if c["cap"] > 0:
        capped = c["cap"] * torch.tanh(capped / c["cap"])
    far = (tq[rq][:, :, None] - s["samples"][:, 3][rk][:, None, :]).abs()
    seen = there_q[:, :, None] & there_k[:, None, :]
    if c["causal"]:
        a = torch.arange(rq.shape[1], device=DEV)[None, :, None] + (s["counts"] - nq)[:, None, None]
        b = torch.arange(rk.shape[1], device=DEV)[None, None, :]
        before = b <= a
        if s["prefix"] is not None:
            before = before | (b < s["prefix"][:, None, None])
        seen = seen & before
    x = torch.where(seen[:, None], capped - s["slopes"][None, :, None, None] * far[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p, v)
    lse = (top + torch.log(total))[..., 0]

    def packed(y, rows, there, like, heads):  # [R, H, L, D] -> [N, heads, D], heads that share one summed
        y = y.view(y.shape[0], heads, -1, *y.shape[2:]).sum(2).transpose(1, 2)
        out = torch.zeros(like.shape[0], heads, y.shape[3], device=DEV)
        out[rows[there]] = y[there]
        return out

    o_rows = packed(o, rq, there_q, s["q"], H).to(s["q"].dtype)
    lse_rows = packed(lse[..., None], rq, there_q, s["q"], H)[..., 0]
    if not c["train"]:
        return o_rows, lse_rows
    do = rays(s["do"], rq)
    dv = torch.matmul(p.transpose(2, 3), do)
    dx = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(-1, keepdim=True))
    if c["cap"] > 0:
        dx = dx * (1.0 - (capped / c["cap"]).square())
    dx = dx * scale
    dq, dk = torch.matmul(dx, k), torch.matmul(dx.transpose(2, 3), q)
    ty = s["q"].dtype
    return (o_rows, lse_rows, packed(dq, rq, there_q, s["q"], H).to(ty), packed(dk, rk, there_k, s["k"], G).to(ty),
            packed(dv, rk, there_k, s["v"], G).to(ty))


def _doubling(a, b, place, longest, step):
    """y_t = a_t y_{t - step} + b_t within each ray; place: steps since its first sample in that direction."""
    rows = torch.arange(a.shape[0], device=DEV)
    d = 1
    while d < longest:
        inside = (place >= d)[:, None]
        src = torch.where(place >= d, rows - step * d, rows)
        b = torch.where(inside, b + a * b[src], b)
        a = torch.where(inside, a * a[src], a)
        d *= 2
    return b


def _scan(s):
    c = s["case"]
    if own:
        import ray_ops
        rays = ray_ops.RaySet(s["counts"], s["offsets"], s["ray_ids"])
        if not c["train"]:
            return ray_ops.ray_scan(s["gate"], s["x"], rays, h0=s["h0"], reverse=c["reverse"])[:2]
        h, last, marks = ray_ops.ray_scan(s["gate"], s["x"], rays, h0=s["h0"], reverse=c["reverse"], marks=True)
        dgate, dx, dh0 = ray_ops.ray_scan_backward(s["dh"], s["gate"], s["x"], marks, rays, dlast=s["dlast"],
                                                   h0=s["h0"], reverse=c["reverse"])
        return (h, last, dgate, dx) + ((dh0,) if c["start"] else ())
    ids, counts, offsets = s["ray_ids"].long(), s["counts"].long(), s["offsets"].long()
    step = -1 if c["reverse"] else 1
    ahead = torch.arange(s["n"], device=DEV) - offsets[ids]
    behind = counts[ids] - 1 - ahead
    place, left = (behind, ahead) if c["reverse"] else (ahead, behind)
    some = counts > 0
    first = torch.where(some, offsets + (counts - 1 if c["reverse"] else 0), 0)
    final = torch.where(some, offsets + (0 if c["reverse"] else counts - 1), 0)
    gate, x = s["gate"].float(), s["x"].float()
    z = torch.sigmoid(gate)
    keep = torch.sigmoid(-gate)
    start = s["h0"] if c["start"] else torch.zeros(c["rays"], c["channels"], device=DEV)
    entering = (place == 0)[:, None]
    h = _doubling(keep, z * x + torch.where(entering, keep * start[ids], 0.0), place, s["longest"], step)
    last = torch.where(some[:, None], h[final], start)
    if not c["train"]:
        return h.to(s["x"].dtype), last
    rows = torch.arange(s["n"], device=DEV)
    ending = (left == 0)[:, None]
    after = torch.where(left > 0, rows + step, rows)
    dh = s["dh"].float() + torch.where(ending, s["dlast"][ids], 0.0)
    g = _doubling(torch.where(ending, 0.0, keep[after]), dh, left, s["longest"], -step)
    before = torch.where(entering, start[ids], h[torch.where(place > 0, rows - step, rows)])
    dgate = g * (x - before) * z * keep
    dh0 = torch.where(some[:, None], (keep * g)[first], s["dlast"])
    ty = s["x"].dtype
    return (h.to(ty), last, dgate.to(ty), (g * z).to(ty)) + ((dh0,) if c["start"] else ())


def _experts(s):
    c = s["case"]
    if own:
        import ray_ops
        plan = ray_ops.expert_plan(s["ids"], c["experts"])
        if c["train"]:
            return ray_ops.expert_linear_backward(s["dy"], s["x"], s["W"], plan, y=s["y"] if c["relu"] else None)
        y = ray_ops.expert_linear(s["x"], s["W"], s["b"], plan, relu=c["relu"])
        return y, plan.counts, plan.rows
    E, most = c["experts"], s["most"]
    rows = torch.sort(s["ids"], stable=True)[1]
    counts = torch.bincount(s["ids"], minlength=E)
    offsets = torch.cumsum(counts, 0) - counts
    at, there = _padded(counts, offsets, most)
    src = rows[at]
    x = s["x"][src].float() * there[..., None]
    W = s["W"].float()
    if not c["train"]:
        y = torch.baddbmm(s["b"].float()[:, None], x, W.transpose(1, 2))
        y = y.clamp(min=0.0) if c["relu"] else y
        out = torch.zeros(c["rows"], c["out"], device=DEV)
        out[src[there]] = y[there]
        return out.to(s["x"].dtype), counts.to(torch.int32), rows.to(torch.int32)
    dy = s["dy"].float()
    dy = torch.where(s["y"] > 0, dy, 0.0) if c["relu"] else dy
    dy = dy[src] * there[..., None]
    dx = torch.zeros(c["rows"], c["k"], device=DEV)
    dx[src[there]] = torch.bmm(dy, W)[there]
    return dx.to(s["x"].dtype), torch.bmm(dy.transpose(1, 2), x), dy.sum(1)


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def exact(c, seed):
    s = prepare(c, seed)
    return {"attention": _exact_attention, "scan": _exact_scan, "experts": _exact_experts}[c["op"]](c, s)


def _exact_attention(c, s):
    """Rays of one length at a time, gradients by automatic differentiation."""
    H, G, D = c["heads"], c["kv_heads"], c["dim"]
    Q = s["q"].shape[0]
    f64 = dict(device=DEV, dtype=torch.float64)
    o, lse = torch.zeros(Q, H, D, **f64), torch.full((Q, H), -math.inf, **f64)
    dq, dk, dv = torch.zeros(Q, H, D, **f64), torch.zeros(s["n"], G, D, **f64), torch.zeros(s["n"], G, D, **f64)
    tk = s["samples"][:, 3].double()
    tq = tk if c["query"] == "all" else s["tq"].double()
    heads = torch.arange(H, device=DEV) // (H // G)
    counts = s["counts"].long()
    for L in torch.unique(counts).tolist():
        if L == 0:
            continue
        every = torch.nonzero(counts == L)[:, 0]
        for which in every.split(max(1, int(4e8 // (H * L * L)))):
            kr = s["offsets"].long()[which][:, None] + torch.arange(L, device=DEV)
            qr = kr if c["query"] == "all" else which[:, None]
            q, k, v = (x.double().requires_grad_(c["train"]) for x in (s["q"][qr], s["k"][kr], s["v"][kr]))
            sc = (q.transpose(1, 2) @ k[:, :, heads].permute(0, 2, 3, 1)) / math.sqrt(D)
            if c["cap"] > 0:
                sc = torch.tanh(sc / c["cap"]) * c["cap"]
            sc = sc - s["slopes"].double()[:, None, None] * (tq[qr][:, None, :, None] - tk[kr][:, None, None, :]).abs()
            if c["causal"]:
                b = torch.arange(L, device=DEV)
                ok = b[None, :] <= b[L - qr.shape[1]:, None]
                ok = ok.expand(len(which), -1, -1)
                if s["prefix"] is not None:
                    ok = ok | (b < s["prefix"][which][:, None])[:, None, :]
                sc = sc.masked_fill(~ok[:, None], -math.inf)
            z = torch.logsumexp(sc, -1)
            y = (torch.softmax(sc, -1) @ v[:, :, heads].transpose(1, 2)).transpose(1, 2)
            if c["train"]:
                gq, gk, gv = torch.autograd.grad(y, (q, k, v), s["do"][qr].double())
                dq[qr], dk[kr], dv[kr] = gq, gk, gv
            o[qr], lse[qr] = y.detach(), z.detach().transpose(1, 2)
            del q, k, v, sc, z, y
    return (o, lse, dq, dk, dv) if c["train"] else (o, lse)


def _exact_scan(c, s):
    """One step of every ray at a time, the longest rays first."""
    counts, offsets = s["counts"].long(), s["offsets"].long()
    by = torch.argsort(counts, descending=True)
    n = counts[by].cpu().numpy()
    first = offsets[by] + (counts[by] - 1).clamp(min=0) if c["reverse"] else offsets[by]
    step, R, C = (-1 if c["reverse"] else 1), c["rays"], c["channels"]
    f64 = dict(device=DEV, dtype=torch.float64)
    state = s["h0"].double()[by] if c["start"] else torch.zeros(R, C, **f64)
    h = torch.zeros(s["n"], C, **f64)
    live = [int(np.searchsorted(-n, -t, side="left")) for t in range(int(n[0]))]  # rays longer than t
    prev = torch.zeros(s["n"], C, **f64) if c["train"] else None
    for t, m in enumerate(live):
        r = first[:m] + step * t
        z = torch.sigmoid(s["gate"][r].double())
        if c["train"]:
            prev[r] = state[:m]
        state[:m] += z * (s["x"][r].double() - state[:m])
        h[r] = state[:m]
    last = torch.empty_like(state)
    last[by] = state
    if not c["train"]:
        return h, last
    d = s["dlast"].double()[by]
    dgate, dx = torch.zeros(s["n"], C, **f64), torch.zeros(s["n"], C, **f64)
    for t in range(len(live) - 1, -1, -1):
        m = live[t]
        r = first[:m] + step * t
        z = torch.sigmoid(s["gate"][r].double())
        d[:m] += s["dh"][r].double()
        dx[r] = z * d[:m]
        dgate[r] = d[:m] * (s["x"][r].double() - prev[r]) * z * (1.0 - z)
        d[:m] *= 1.0 - z
    dh0 = torch.empty_like(d)
    dh0[by] = d
    return (h, last, dgate, dx) + ((dh0,) if c["start"] else ())


def _exact_experts(c, s):
    """One expert at a time."""
    out = torch.zeros(c["rows"], c["k"] if c["train"] else c["out"], device=DEV, dtype=torch.float64)
    dW, db = [], []
    for e in range(c["experts"]):
        r = torch.nonzero(s["ids"] == e)[:, 0]
        x, W = s["x"][r].double(), s["W"][e].double()
        if c["train"]:
            g = s["dy"][r].double()
            if c["relu"]:
                g = g * (s["y"][r] > 0)
            out[r] = g @ W
            dW.append(g.T @ x)
            db.append(g.sum(0))
        else:
            y = x @ W.T + s["b"][e].double()
            out[r] = torch.relu(y) if c["relu"] else y
    return (out, torch.stack(dW), torch.stack(db)) if c["train"] else (out, None, None)
