"""Blocks of a model along rays, as cases that can be timed and checked: norm, memory, routing to several experts.

A block takes the packed samples that `ffn_march` leaves (`counts`, `offsets` per ray, `ray_ids` per sample), normalises
their features, lets each ray carry a matrix of what its samples have shown, and blends the layers of several experts:

  norm    y = (x - mean) / sqrt(var + eps) * weight + bias by rows, and its gradients
  delta   a state S [dk, dv] a ray and head: S_t = a_t S_{t-1} + k_t n_t^T with n_t = b_t (v_t - a_t S_{t-1}^T k_t) and
          a_t = exp(decay_t), read as o_t = scale S_t^T q_t; a whole batch, a ray's next sample, and the gradients
  route   every row goes to k experts: copies of the rows in the experts' order, and the weighted sums back

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
EPS = 1e-5
CHUNK = 64  # rows whose products the plain form of delta takes at once, where rays are that long


# ---------------------------------------------------------------------------
# the cases


def listed() -> list:
    return [
        # the samples of an interactive pick's two rays before a layer: the launch is all of it
        dict(name="norm_few", op="norm", rows=37, width=64, type="bf16", params="fp32", bias=True, train=False),
        # a marched training step's batch, the width of the ray model's features
        dict(name="norm_batch_train", op="norm", rows=1 << 22, width=64, type="bf16", params="fp32", bias=True,
             train=True),
        # a wide trunk, parameters in the rows' own type
        dict(name="norm_wide_train", op="norm", rows=20011, width=4096, type="bf16", params="bf16", bias=True,
             train=True),
        # the framework's default arithmetic, rows that fill no line, no bias
        dict(name="norm_odd_train", op="norm", rows=100003, width=333, type="fp32", params="fp32", bias=False,
             train=True),
        # one more sample of each of a preview's rays: the states go through once and little else does
        dict(name="delta_step", op="delta", rays=2048, mean=0, longest=1, spread="even", heads=4, v_heads=4, dk=64,
             dv=64, type="bf16", reverse=False, start=True, last=True, train=False),
        # a training batch of the marched step's kind: short rays of every length
        dict(name="delta_train", op="delta", rays=8192, mean=28, longest=256, spread="marched", heads=4, v_heads=4,
             dk=32, dv=32, type="bf16", reverse=False, start=False, last=False, train=True),
        # few long rays, two value heads on a key head: the rows of a ray are one chain
        dict(name="delta_long_train", op="delta", rays=24, mean=0, longest=4096, spread="even", heads=4, v_heads=8,
             dk=64, dv=64, type="bf16", reverse=False, start=False, last=False, train=True),
        # the framework's default arithmetic, odd sizes, back to front as compositing goes, from a state and to one
        dict(name="delta_odd_train", op="delta", rays=3001, mean=40, longest=200, spread="marched", heads=3, v_heads=3,
             dk=24, dv=40, type="fp32", reverse=True, start=True, last=True, train=True),
        # a pick's samples to two of a scene's regions
        dict(name="route_few", op="route", rows=24, k=2, experts=8, width=64, skew=1.0, dropped=0.0, type="fp32",
             train=False),
        # a marched batch's samples, each to its own region and the nearest other one
        dict(name="route_batch", op="route", rows=1 << 20, k=2, experts=64, width=64, skew=1.0, dropped=0.02,
             type="bf16", train=False),
        # blending over the eight corners of a cell: many narrow rows, and the gradients
        dict(name="route_corners_train", op="route", rows=300007, k=8, experts=27, width=32, skew=0.7, dropped=0.0,
             type="fp16", train=True),
        # wide rows to four of many experts, some of them empty, a tenth of the places past their experts' capacity
        dict(name="route_wide_train", op="route", rows=50021, k=4, experts=128, width=1024, skew=1.0, dropped=0.1,
             type="bf16", train=True),
    ]


def _log(rng, lo, hi) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["norm", "delta", "delta", "route"])
    ty = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "norm":
        width = rng.choice([_log(rng, 5, 8192), 8 * _log(rng, 1, 1024), 64, 128])
        return dict(op=op, rows=_log(rng, 1, int(2.0e8 / max(width, 16))), width=width, type=ty,
                    params=rng.choice(["fp32", ty]), bias=rng.random() < 0.7, train=rng.random() < 0.7)
    if op == "route":
        k, width = rng.choice([1, 2, 2, 3, 4, 8]), rng.choice([8, 16, 32, 64, 72, 128, 256, 1024])
        return dict(op=op, rows=_log(rng, 1, int(min(2 << 20, 1.0e8 / (k * width)))), k=k, experts=_log(rng, k, 256),
                    width=width, skew=rng.choice([0.0, 0.7, 1.5]), dropped=rng.choice([0.0, 0.0, 0.1]), type=ty,
                    train=rng.random() < 0.5)
    heads, share = rng.choice([1, 2, 3, 4]), rng.choice([1, 1, 2])
    c = dict(op=op, rays=0, mean=0, longest=0, spread="even", heads=heads, v_heads=heads * share,
             dk=rng.choice([16, 24, 32, 64, 64, 128]), dv=rng.choice([16, 32, 40, 64, 64, 128]), type=ty,
             reverse=rng.random() < 0.3, start=rng.random() < 0.5, last=rng.random() < 0.5, train=False)
    states = c["v_heads"] * c["dk"] * c["dv"]
    if rng.random() < 0.25:  # a ray's next sample, or its next few
        c["longest"], c["start"], c["last"] = rng.choice([1, 1, 2, 3]), True, True
        c["rays"] = _log(rng, 1, int(min(16384, 1.0e8 / (states * c["longest"]))))
        return c
    c["train"], c["longest"] = rng.random() < 0.6, _log(rng, 16, 4096)
    # the rows of a padded batch, and the states that pass, stay under those of the largest listed case
    c["rays"] = _log(rng, 1, int(max(1, min(8192, 2.4e9 / (c["longest"] * states),
                                            5.0e7 / (c["longest"] * c["v_heads"] * max(c["dk"], c["dv"]) / 64)))))
    if c["rays"] >= 64 and rng.random() < 0.7:
        c["spread"], c["mean"] = "marched", max(2, c["longest"] // rng.choice([2, 4, 8]))
    return c


def _fixed(c) -> np.random.RandomState:
    """Lengths go by the case alone, so that `work` knows them."""
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


def work(c) -> dict:
    b = 4 if c["type"] == "fp32" else 2
    if c["op"] == "norm":
        n, w, p = c["rows"], c["width"], (4 if c["params"] == "fp32" else b)
        params = p * w * (2 if c["bias"] else 1)
        if c["train"]:  # x, dy in; y, dx, dweight, dbias out
            return {"bytes": float(4 * b * n * w + 8 * n + params + 8 * w), "flops": 20.0 * n * w}
        return {"bytes": float(2 * b * n * w + 8 * n + params), "flops": 8.0 * n * w}
    if c["op"] == "route":
        n, k, w = c["rows"], c["k"], c["width"]
        bytes_ = b * w * (2 * n + 2 * n * k) + 4 * n * k * 4 + 4 * c["experts"]  # ids, weights, slots, rows; x, xs, y, out
        flops = 2.0 * n * k * w
        if c["train"]:  # dout, dxs in; dy, dx, dweights out
            bytes_ += b * w * (2 * n + 2 * n * k) + 4 * n * k
            flops *= 4
        return {"bytes": float(bytes_), "flops": flops}
    N, R, H, G, dk, dv = float(lengths(c).sum()), c["rays"], c["heads"], c["v_heads"], c["dk"], c["dv"]
    bytes_ = N * b * (2 * H * dk + 2 * G * dv + 2 * G) + 4.0 * R * G * dk * dv * (c["start"] + c["last"])
    flops = 6.0 * N * G * dk * dv
    if c["train"]:  # do in; dq, dk, dv, ddecay, dbeta out; gradients of the states
        bytes_ += N * b * (2 * H * dk + 2 * G * dv + 2 * G) + 4.0 * R * G * dk * dv * (c["start"] + c["last"])
        flops *= 3
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------
# inputs


def prepare(c, seed) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    ty = TYPES[c["type"]]

    def normal(*shape, dtype=ty, scale=1.0, shift=0.0):
        x = torch.empty(shape, device=DEV, dtype=torch.float32).normal_(shift, scale, generator=gen)
        return x.to(dtype)

    if c["op"] == "norm":
        n, w, pt = c["rows"], c["width"], TYPES[c["params"]]
        s = dict(case=c, weight=normal(w, dtype=pt, scale=0.2, shift=1.0),
                 bias=normal(w, dtype=pt, scale=0.1) if c["bias"] else None)
        s["x"] = normal(n, w, shift=0.5)  # features have a mean of their own
        if c["train"]:
            s["dy"] = normal(n, w)
        return s
    if c["op"] == "route":
        n, k, E, w = c["rows"], c["k"], c["experts"], c["width"]
        r = _fixed(c)
        p = (1.0 + np.arange(E)) ** -c["skew"] * (0.5 + r.rand(E))
        if E >= 10 * k:
            p[r.permutation(E)[:E // 10]] = 0.0
        # k different experts a row, the likeliest first: the largest of log p with noise, as a router's scores give them
        score = torch.from_numpy(np.log(np.maximum(p, 1e-30))).to(DEV, torch.float32)
        noise = torch.empty(n, E, device=DEV).exponential_(generator=gen).log_().neg_()
        top, ids = torch.topk(score + noise, k, dim=1)
        ids = ids.to(torch.int32)
        if c["dropped"]:
            ids = torch.where(torch.rand(n, k, device=DEV, generator=gen) < c["dropped"], -1, ids)
        s = dict(case=c, ids=ids.contiguous(), weights=torch.softmax(top, 1).contiguous(), x=normal(n, w),
                 y=normal(n * k, w))
        if c["train"]:
            s["dout"], s["dxs"] = normal(n, w), normal(n * k, w)
        return s
    n = lengths(c)
    n = n[np.random.RandomState(int(seed) & 0x7FFFFFFF).permutation(len(n))]
    N, R, H, G = int(n.sum()), len(n), c["heads"], c["v_heads"]
    counts = torch.from_numpy(n).to(DEV)
    offsets = torch.cumsum(counts, 0) - counts
    s = dict(case=c, n=N, longest=c["longest"], counts=counts.to(torch.int32), offsets=offsets.to(torch.int32),
             ray_ids=torch.repeat_interleave(torch.arange(R, device=DEV), counts).to(torch.int32))

    def unit(*shape):  # keys and queries of length 1
        x = normal(*shape, dtype=torch.float32)
        return (x / x.square().sum(-1, keepdim=True).sqrt()).to(ty)

    s["q"], s["k"], s["v"] = unit(N, H, c["dk"]), unit(N, H, c["dk"]), normal(N, G, c["dv"])
    # states that last some tens of rows, some heads' far longer; writes of every strength
    s["decay"] = (-torch.log1p(normal(N, G, dtype=torch.float32, scale=1.5, shift=-3.5).exp())).to(ty)
    s["beta"] = torch.sigmoid(normal(N, G, dtype=torch.float32)).to(ty)
    s["h0"] = normal(R, G, c["dk"], c["dv"], dtype=torch.float32) if c["start"] else None
    if c["train"]:
        s["do"] = normal(N, G, c["dv"])
        s["dlast"] = normal(R, G, c["dk"], c["dv"], dtype=torch.float32) if c["last"] else None
    return s


# ---------------------------------------------------------------------------
# one pass


def run(s):
    return {"norm": _norm, "delta": _delta, "route": _route}[s["case"]["op"]](s)


def _norm(s):
    c, x, weight, bias = s["case"], s["x"], s["weight"], s["bias"]
    if own:
        import ray_ops
        y, mean, rstd = ray_ops.layer_norm(x, weight, bias, eps=EPS)
        if not c["train"]:
            return y, mean, rstd
        return (y, mean, rstd) + tuple(ray_ops.layer_norm_backward(s["dy"], x, weight, mean, rstd))
    xf, w = x.float(), weight.float()
    mean = xf.mean(1, keepdim=True)
    d = xf - mean
    rstd = 1.0 / torch.sqrt(d.square().mean(1, keepdim=True) + EPS)
    xhat = d * rstd
    y = xhat * w
    if bias is not None:
        y = y + bias.float()
    out = (y.to(x.dtype), mean[:, 0], rstd[:, 0])
    if not c["train"]:
        return out
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return out + (dx.to(x.dtype), (dy * xhat).sum(0), dy.sum(0))


def _route(s):
    c, x, y, ids, weights = s["case"], s["x"], s["y"], s["ids"], s["weights"]
    if own:
        import ray_ops
        route = ray_ops.expert_route(ids, c["experts"])
        out = (route.plan.counts, route.plan.rows, route.slots, ray_ops.expert_dispatch(x, route),
               ray_ops.expert_combine(y, route, weights))
        if not c["train"]:
            return out
        return out + tuple(ray_ops.expert_combine_backward(s["dout"], y, route, weights)) + (
            ray_ops.expert_dispatch_backward(s["dxs"], route),)
    n, k, E = c["rows"], c["k"], c["experts"]
    flat = ids.reshape(-1).long()
    there = (flat >= 0) & (flat < E)
    rows = torch.sort(torch.where(there, flat, E), stable=True)[1]  # place i * k + j is row i's j-th expert
    counts = torch.bincount(flat[there], minlength=E)
    slots = torch.empty_like(rows)
    slots[rows] = torch.arange(n * k, device=DEV)
    kept = there[rows][:, None]
    xs = torch.where(kept, x[rows // k], 0)
    w = torch.where(there.view(n, k), weights, 0.0)
    yk = torch.where(there[:, None], y[slots].float(), 0.0).view(n, k, -1)
    total = (w[:, :, None] * yk).sum(1)
    out = (counts.to(torch.int32), rows.to(torch.int32), slots.view(n, k).to(torch.int32), xs, total.to(x.dtype))
    if not c["train"]:
        return out
    dout = s["dout"].float()
    dy = torch.where(kept, w.reshape(-1)[rows][:, None] * dout[rows // k], 0.0)
    dw = (dout[:, None, :] * yk).sum(2)
    dx = torch.where(there[:, None], s["dxs"][slots].float(), 0.0).view(n, k, -1).sum(1)
    return out + (dy.to(x.dtype), dw, dx.to(x.dtype))


def _inverse(A):
    """(I + A)^-1 of strictly lower triangular A [..., m, m], m a power of two, by halves."""
    m = A.shape[-1]
    if m == 1:
        return torch.ones_like(A)
    h = m // 2
    a, b = _inverse(A[..., :h, :h]), _inverse(A[..., h:, h:])
    low = -torch.matmul(b, torch.matmul(A[..., h:, :h], a))
    return torch.cat((torch.cat((a, torch.zeros_like(a)), -1), torch.cat((low, b), -1)), -2)


def _delta_padded(q, k, v, decay, beta, state, chunk, scale):
    """o and the last state of padded rays: q, k [R, G, L, dk], v [R, G, L, dv], decay, beta [R, G, L], L of whole chunks.
    What a chunk's rows do to each other is taken for all chunks at once; the state passes from chunk to chunk."""
    R, G, L = decay.shape
    n = L // chunk
    q, k, v = (x.reshape(R, G, n, chunk, -1) for x in (q, k, v))
    g = decay.double().reshape(R, G, n, chunk).cumsum(-1)  # differences of long sums
    beta = beta.reshape(R, G, n, chunk, 1)
    lower = torch.ones(chunk, chunk, device=DEV, dtype=torch.bool).tril()
    between = torch.where(lower, g[..., :, None] - g[..., None, :], -math.inf).exp().float()
    since, left = g.exp().float()[..., None], (g[..., -1:] - g).exp().float()[..., None]
    kt = k.transpose(-1, -2)
    T = _inverse((beta * between * torch.matmul(k, kt)).tril(-1))
    U, W = torch.matmul(T, beta * v), torch.matmul(T, beta * since * k)
    P = scale * between * torch.matmul(q, kt)
    qs, ke = scale * since * q, (left * k).transpose(-1, -2)
    o = []
    for i in range(n):
        new = U[:, :, i] - torch.matmul(W[:, :, i], state)
        o.append(torch.matmul(qs[:, :, i], state) + torch.matmul(P[:, :, i], new))
        state = since[:, :, i, -1:] * state + torch.matmul(ke[:, :, i], new)
    return torch.cat(o, 2), state


def _delta(s):
    c = s["case"]
    if own:
        import ray_ops
        rays = ray_ops.RaySet(s["counts"], s["offsets"], s["ray_ids"])
        x = (s["q"], s["k"], s["v"], s["decay"], s["beta"])
        opt = dict(h0=s["h0"], reverse=c["reverse"])
        o, last, marks = ray_ops.ray_delta(*x, rays, last=c["last"], marks=c["train"], **opt)
        out = (o,) + ((last,) if c["last"] else ())
        if not c["train"]:
            return out
        grads = ray_ops.ray_delta_backward(s["do"], *x, marks, rays, dlast=s["dlast"], **opt)
        return out + tuple(grads[:5]) + ((grads[5],) if c["start"] else ())
    H, G, R = c["heads"], c["v_heads"], c["rays"]
    counts, offsets = s["counts"].long()[:, None], s["offsets"].long()[:, None]
    chunk = min(CHUNK, 1 << (s["longest"] - 1).bit_length())
    L = -(-s["longest"] // chunk) * chunk
    at = torch.arange(L, device=DEV)
    there = at < counts
    rows = torch.where(there, offsets + (counts - 1 - at if c["reverse"] else at), 0)
    # rows past a ray's end write nothing and leave the state as it is
    padded = []
    for m in ("q", "k", "v", "decay", "beta"):
        x = s[m]
        x = torch.where(there.view(R, L, *[1] * (x.dim() - 1)), x[rows].float(), 0.0)
        padded.append(x.repeat_interleave(G // x.shape[2], 2).transpose(1, 2).contiguous().requires_grad_(c["train"]))
    h0 = s["h0"] if c["start"] else torch.zeros(R, G, c["dk"], c["dv"], device=DEV)
    padded.append(h0.detach().requires_grad_(c["train"]))
    with torch.set_grad_enabled(c["train"]):
        y, last = _delta_padded(*padded, chunk, c["dk"] ** -0.5)
    ty = s["q"].dtype

    order = rows[there]

    def back(x, heads):  # [R, G, L, ...] -> [N, heads, ...], heads that share one summed
        x = x.transpose(1, 2)[there]
        out = torch.empty(s["n"], heads, *x.shape[2:], device=DEV)
        out[order] = x.view(s["n"], heads, G // heads, *x.shape[2:]).sum(2)
        return out.to(ty)

    out = (back(y.detach(), G),) + ((last.detach(),) if c["last"] else ())
    if not c["train"]:
        return out
    dy = torch.where(there[:, :, None, None], s["do"][rows].float(), 0.0).transpose(1, 2)
    grads = torch.autograd.grad((y, last) if c["last"] else (y,), padded, (dy, s["dlast"]) if c["last"] else (dy,))
    return out + tuple(back(x, heads) for x, heads in zip(grads, (H, H, G, G, G))) + ((grads[5],) if c["start"] else ())


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def exact(c, seed):
    s = prepare(c, seed)
    return {"norm": _exact_norm, "delta": _exact_delta, "route": _exact_route}[c["op"]](c, s)


def _exact_norm(c, s):
    """Gradients from those of the mean and of the variance."""
    x, w = s["x"].double(), s["weight"].double()
    n = c["width"]
    mean = x.sum(1) / n
    var = (x - mean[:, None]).pow(2).sum(1) / n
    rstd = (var + EPS) ** -0.5
    xc = x - mean[:, None]
    y = xc * rstd[:, None] * w + (s["bias"].double() if c["bias"] else 0.0)
    if not c["train"]:
        return y, mean, rstd
    dy = s["dy"].double()
    g = dy * w
    dvar = -0.5 * (g * xc).sum(1) * rstd ** 3
    dmean = -(g.sum(1) * rstd) - 2.0 * dvar * xc.sum(1) / n
    dx = g * rstd[:, None] + (2.0 * dvar / n)[:, None] * xc + (dmean / n)[:, None]
    return y, mean, rstd, dx, (dy * xc * rstd[:, None]).sum(0), dy.sum(0)


def _exact_route(c, s):
    """One of a row's places at a time; a place's slot is the number of places before it in the order of (expert, place)."""
    n, k, E = c["rows"], c["k"], c["experts"]
    ids = s["ids"].long()
    inside = (ids >= 0) & (ids < E)
    place = torch.arange(n * k, device=DEV).view(n, k)
    key = torch.where(inside, ids, E) * (n * k) + place
    order = torch.argsort(key.view(-1))
    slot = torch.searchsorted(key.view(-1)[order], key)
    total = torch.zeros(n, c["width"], device=DEV, dtype=torch.float64)
    xs = torch.zeros(n * k, c["width"], device=DEV, dtype=torch.float64)
    dy, dx = torch.zeros_like(xs), torch.zeros_like(total)
    dw = torch.zeros(n, k, device=DEV, dtype=torch.float64)
    for j in range(k):
        i = torch.nonzero(inside[:, j])[:, 0]
        at, w = slot[i, j], s["weights"][i, j].double()[:, None]
        xs[at] = s["x"][i].double()
        y = s["y"][at].double()
        total[i] += w * y
        if c["train"]:
            dout = s["dout"][i].double()
            dy[at] = w * dout
            dw[i, j] = (dout * y).sum(1)
            dx[i] += s["dxs"][at].double()
    return (None, None, None, xs, total) + ((dy, dw, dx) if c["train"] else ())


def _exact_delta(c, s):
    """One row of every ray at a time, the longest rays first; gradients row by row, back again."""
    H, G, R, dk, dv = c["heads"], c["v_heads"], c["rays"], c["dk"], c["dv"]
    counts, offsets = s["counts"].long(), s["offsets"].long()
    by = torch.argsort(counts, descending=True)
    n = counts[by].cpu().numpy()
    first = offsets[by] + (counts[by] - 1).clamp(min=0) if c["reverse"] else offsets[by]
    step, scale = (-1 if c["reverse"] else 1), 1.0 / math.sqrt(dk)
    f64 = dict(device=DEV, dtype=torch.float64)
    of = torch.arange(G, device=DEV) // (G // H)  # the key head of each value head
    S = s["h0"].double()[by] if c["start"] else torch.zeros(R, G, dk, dv, **f64)
    live = [int(np.searchsorted(-n, -t, side="left")) for t in range(int(n[0]))]  # rays longer than t

    def rows(t, m):
        r = first[:m] + step * t
        q, k = s["q"][r][:, of].double(), s["k"][r][:, of].double()
        a = s["decay"][r].double().exp()[..., None, None]
        return r, q, k, s["v"][r].double(), a, s["beta"][r].double()[..., None]

    o = torch.zeros(s["n"], G, dv, **f64)
    kept = []
    for t, m in enumerate(live):
        r, q, k, v, a, b = rows(t, m)
        if c["train"]:
            kept.append(S[:m].clone())
        S1 = a * S[:m]
        new = b * (v - (k[..., None] * S1).sum(-2))
        S1 += k[..., None] * new[..., None, :]
        o[r] = scale * (q[..., None] * S1).sum(-2)
        S[:m] = S1
    last = torch.empty_like(S)
    last[by] = S
    out = (o,) + ((last,) if c["last"] else ())
    if not c["train"]:
        return out
    D = s["dlast"].double()[by] if c["last"] else torch.zeros_like(S)
    dq, dkey = torch.zeros(s["n"], H, dk, **f64), torch.zeros(s["n"], H, dk, **f64)
    dval, dg, db = torch.zeros(s["n"], G, dv, **f64), torch.zeros(s["n"], G, **f64), torch.zeros(s["n"], G, **f64)
    for t in range(len(live) - 1, -1, -1):
        m = live[t]
        r, q, k, v, a, b = rows(t, m)
        do = s["do"][r].double()
        S0 = a * kept.pop()
        u = v - (k[..., None] * S0).sum(-2)
        S1 = S0 + k[..., None] * (b * u)[..., None, :]
        D1 = D[:m] + scale * q[..., None] * do[..., None, :]
        dnew = (k[..., None] * D1).sum(-2)
        du = b * dnew
        D0 = D1 - k[..., None] * du[..., None, :]
        grad_k = (D1 * (b * u)[..., None, :]).sum(-1) - (S0 * du[..., None, :]).sum(-1)
        grad_q = scale * (S1 * do[..., None, :]).sum(-1)
        dq[r] = grad_q.view(m, H, G // H, dk).sum(2)
        dkey[r] = grad_k.view(m, H, G // H, dk).sum(2)
        dval[r], db[r], dg[r] = du, (dnew * u).sum(-1), (D0 * S0).sum((-1, -2))
        D[:m] = a * D0
    dh0 = torch.empty_like(D)
    dh0[by] = D
    return out + (dq, dkey, dval, dg, db) + ((dh0,) if c["start"] else ())
