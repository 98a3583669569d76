"""The delta rule's values and gradients as a whole, ray by ray and head by head, against 64 bits: bounds that go by the gradient.

A result of the type is off by half a step at most, eps / 2 of itself, and by what float operands make of its terms before that.
Those are products of a row's vectors with the states before it and their gradients: each is known to some 2^-22 of its size
(states that hold some hundred rounded products, none of which grows: see delta_oracle), and errors of neighbouring rows differ.
2^-19 of the sizes' norm is allowed.  A decay's gradient is the sum of such terms from its row to its chunk's end, 16 rows at
most, and the states' product there: it is known to its terms' sizes, not to its own where they cancel."""
from __future__ import annotations

import torch

from delta_oracle import Delta, inputs
from ray_oracle import F64, TINY, ray_set

NAMES = ("o", "last", "dq", "dk", "dv", "ddecay", "dbeta", "dh0")

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32
# lens, H, G, dk, dv, type, keys, reverse, start
CASES = [
    ([37, 5, 0, 16], 2, 2, 32, 32, BF, "random", False, True), ([37, 5, 0, 16], 2, 2, 32, 32, FL, "random", True, False),
    ([37, 5, 0, 16], 1, 3, 24, 40, HF, "random", False, True), ([33, 64, 31], 1, 2, 64, 64, BF, "random", True, True),
    ([33, 64, 31], 1, 1, 128, 128, BF, "random", False, True), ([33, 64, 31], 1, 1, 128, 128, FL, "random", False, False),
    ([33, 20], 1, 1, 128, 128, HF, "random", False, True), ([130, 40], 2, 2, 32, 32, FL, "alike", False, True),
    ([130, 40], 2, 2, 32, 32, BF, "alike", False, True), ([700, 300], 1, 1, 64, 64, FL, "random", False, True),
    ([700, 300], 1, 2, 64, 64, BF, "random", False, False), ([700], 1, 1, 16, 16, HF, "random", True, False),
    ([90, 17], 1, 1, 72, 104, BF, "random", False, True), ([90, 17], 1, 1, 16, 48, BF, "random", False, True),
    ([50, 50], 1, 4, 8, 8, FL, "random", True, True), ([50, 50], 2, 2, 40, 16, BF, "random", True, False),
]


def make(case, seed=0):
    """(rays, [q, k, v, decay, beta], h0, do, dlast)"""
    lens, H, G, dk, dv, dtype, keys, reverse, start = case
    rays = ray_set(lens)
    g = torch.Generator().manual_seed(seed + 50)
    state = (len(lens), G, dk, dv)
    h0, dlast = ((torch.randn(state, generator=g), torch.randn(state, generator=g)) if start else (None, None))
    return rays, inputs(rays[3], H, G, dk, dv, dtype, seed, keys), h0, torch.randn(rays[3], G, dv, generator=g).to(dtype), dlast


def wanted(case, rays, x, h0, do, dlast):
    """{name: (value, size)}, sizes a row and value head (a ray and value head for states)."""
    d = Delta(*x, rays, h0, reverse=case[7])
    n, G = d.n, d.G
    size = {k: torch.zeros(n, G, dtype=F64) for k in ("o", "dq", "dk", "dv", "ddecay", "dbeta")}
    value = {k: torch.zeros(n, G, w, dtype=F64) for k, w in (("dq", d.dk), ("dk", d.dk), ("dv", d.dv))}
    value.update({k: torch.zeros(n, G, dtype=F64) for k in ("ddecay", "dbeta")})
    do = do.to(F64)
    dh0 = torch.zeros(d.last.shape, dtype=F64) if dlast is None else dlast.to(F64).clone()
    size["last"] = torch.zeros(d.last.shape[:2], dtype=F64)
    size["dh0"] = dh0.norm(dim=(-1, -2))

    def norm(t):
        return t.norm(dim=-1)

    for r, rows in enumerate(d.rows):
        D = dh0[r].clone()
        terms = []
        size["last"][r] = d.last[r].norm(dim=(-1, -2))
        for place in range(len(rows) - 1, -1, -1):
            i, S = rows[place], d.kept[r][place]
            q, k, v, a, b = d.q[i], d.k[i], d.v[i], d.a[i], d.b[i]
            S0 = a[:, None, None] * S
            u = v - (k[:, :, None] * S0).sum(1)
            S1 = S0 + k[:, :, None] * (b[:, None] * u)[:, None, :]
            D1 = D + d.scale * q[:, :, None] * do[i][:, None, :]
            dn = (k[:, :, None] * D1).sum(1)
            du = b[:, None] * dn
            D0 = D1 - k[:, :, None] * du[:, None, :]
            s0, s1, d1 = (t.norm(dim=(-1, -2)) for t in (S0, S1, D1))
            su, sn = norm(v) + norm(k) * s0, norm(k) * d1  # of u and dn
            value["dq"][i] = d.scale * (S1 * do[i][:, None, :]).sum(-1)
            value["dk"][i] = (D1 * (b[:, None] * u)[:, None, :]).sum(-1) - (S0 * du[:, None, :]).sum(-1)
            value["dv"][i], value["dbeta"][i], value["ddecay"][i] = du, (dn * u).sum(-1), (D0 * S0).sum((-1, -2))
            size["o"][i] = abs(d.scale) * norm(q) * s1
            size["dq"][i] = abs(d.scale) * s1 * norm(do[i])
            size["dk"][i] = b * (d1 * su + s0 * sn)
            size["dv"][i], size["dbeta"][i] = b * sn, sn * su
            terms.append((i, norm(q) * size["dq"][i] + norm(k) * size["dk"][i], D.norm(dim=(-1, -2)) * s1))
            D = a[:, None, None] * D0
            size["dh0"][r] = torch.maximum(size["dh0"][r], D.norm(dim=(-1, -2)))
        # from each row to its chunk's end (chunks of 16 from the first place on)
        for j, (i, _, _) in enumerate(terms):  # terms[0] is the ray's last place
            place = len(rows) - 1 - j
            end = min(len(rows) - 1, place // 16 * 16 + 15)
            of = terms[len(rows) - 1 - end:j + 1]
            size["ddecay"][i] = torch.stack([t[1] for t in of]).square().sum(0).sqrt() + of[0][2]
        dh0[r] = D
    value.update(o=d.o, last=d.last, dh0=dh0)
    for k in ("dq", "dk"):  # of shared heads
        value[k] = value[k].view(n, d.H, G // d.H, -1).sum(2)
        size[k] = size[k].view(n, d.H, G // d.H).square().sum(2).sqrt()
    return {k: (value[k], size[k]) for k in NAMES if k != "dh0" or h0 is not None}


def off(case, rays, got: dict, want: dict) -> list:
    """[(name, ray, head, off, allowed)] of what is further off than it may be."""
    counts, offsets = rays[0].tolist(), rays[1].tolist()
    bad = []
    for name, t in got.items():
        if t is None:
            continue
        value, size = want[name]
        dtype = FL if name in ("last", "dh0") else case[5]
        diff = (t.detach().cpu().to(F64) - value).reshape(*size.shape, -1)
        value = value.reshape(*size.shape, -1)
        for r, (c, o) in enumerate(zip(counts, offsets)):
            rows = slice(r, r + 1) if name in ("last", "dh0") else slice(o, o + c)
            v, e, s = value[rows], diff[rows], size[rows]
            allowed = (torch.finfo(dtype).eps / 2 * v.norm(dim=(0, 2)) + 2.0 ** -19 * s.norm(dim=0)
                       + TINY[dtype] * v[:, 0].numel() ** 0.5)
            far = e.norm(dim=(0, 2))
            bad += [(name, r, h, float(far[h]), float(allowed[h])) for h in range(size.shape[1]) if not far[h] <= allowed[h]]
    return bad
