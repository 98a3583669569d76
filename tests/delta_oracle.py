"""The delta rule with decay, row by row in 64 bits (CPU), and its gradients, with bounds of the kernel's rounding.

A row's map S -> a (I - b k k^T) S does not lengthen a column of S where b |k|^2 <= 2 and a <= 1, so that an error made in one
chunk of 16 rows is not enlarged by the later ones, and errors of chunks add up at most.  Within a chunk the kernel's
values are sums in float of at most 128 + 16 products, taken four at a time, and a substitution through 15 rows: 128 float
steps of the sizes that enter (a state's column, a value) are allowed for a chunk."""
from __future__ import annotations

import torch

from ray_oracle import F64, TINY, U


class Delta:
    def __init__(self, q, k, v, decay, beta, rays, h0=None, scale=None, reverse=False):
        counts, offsets, _, n = rays
        self.H, self.G, self.dk, self.dv = q.shape[1], v.shape[1], q.shape[2], v.shape[2]
        self.scale = self.dk ** -0.5 if scale is None else scale
        self.of = torch.arange(self.G) // (self.G // self.H)
        self.q, self.k, self.v = q.to(F64)[:, self.of], k.to(F64)[:, self.of], v.to(F64)
        self.a, self.b = decay.to(F64).exp(), beta.to(F64)
        R = len(counts)
        state = (R, self.G, self.dk, self.dv)
        self.last = torch.zeros(state, dtype=F64) if h0 is None else h0.to(F64).clone()
        self.o, self.n = torch.zeros(n, self.G, self.dv, dtype=F64), n
        self.o_size = torch.zeros(n, self.G, self.dv, dtype=F64)
        self.rows, self.kept, self.size = [], [], []  # states before each row; the largest column of S or value of a ray
        for r in range(R):
            o, m = int(offsets[r]), int(counts[r])
            rows = list(range(o, o + m))[::-1] if reverse else list(range(o, o + m))
            S, kept = self.last[r].clone(), []
            size = S.norm(dim=-2)
            for i in rows:
                kept.append(S)
                S0 = self.a[i][:, None, None] * S
                new = self.b[i][:, None] * (self.v[i] - (self.k[i][:, :, None] * S0).sum(1))
                S = S0 + self.k[i][:, :, None] * new[:, None, :]
                self.o[i] = self.scale * (self.q[i][:, :, None] * S).sum(1)
                size = torch.maximum(size, torch.maximum(S.norm(dim=-2), self.v[i].abs()))
            for i in rows:
                self.o_size[i] = abs(self.scale) * self.q[i].norm(dim=-1)[:, None] * size
            self.last[r] = S
            self.rows.append(rows), self.kept.append(kept), self.size.append(size)
        chunks = max([1] + [(len(x) + 15) // 16 for x in self.rows])
        self.eps = 2.0 ** -24 * 128 * chunks

    def bounds(self, dtype):
        last = torch.stack(self.size)[:, :, None, :].expand(self.last.shape) if self.rows else self.last
        return U[dtype] * self.o.abs() + self.eps * self.o_size + TINY[dtype], self.eps * last + 1e-37

    def backward(self, do, dlast, dtype):
        """[(gradient, bound)] of q, k, v, decay, beta, h0."""
        do = do.to(F64)
        n, G = self.n, self.G
        dq, dk = torch.zeros(n, G, self.dk, dtype=F64), torch.zeros(n, G, self.dk, dtype=F64)
        dv, dg, db = torch.zeros(n, G, self.dv, dtype=F64), torch.zeros(n, G, dtype=F64), torch.zeros(n, G, dtype=F64)
        bq, bk, bv, bg, bb = (torch.zeros_like(x) for x in (dq, dk, dv, dg, db))
        dh0 = torch.zeros(self.last.shape, dtype=F64) if dlast is None else dlast.to(F64).clone()
        bh = torch.zeros_like(dh0)
        for r, rows in enumerate(self.rows):
            D, size = dh0[r].clone(), self.size[r]
            gsize = D.norm(dim=-2)
            for i, S in zip(reversed(rows), reversed(self.kept[r])):
                q, k, a, b = self.q[i], self.k[i], self.a[i][:, None, None], self.b[i][:, None]
                S0 = a * S
                u = self.v[i] - (k[:, :, None] * S0).sum(1)
                S1 = S0 + k[:, :, None] * (b * u)[:, None, :]
                D1 = D + self.scale * q[:, :, None] * do[i][:, None, :]
                dn = (k[:, :, None] * D1).sum(1)
                du = b * dn
                D0 = D1 - k[:, :, None] * du[:, None, :]
                dq[i] = self.scale * (S1 * do[i][:, None, :]).sum(-1)
                dk[i] = (D1 * (b * u)[:, None, :]).sum(-1) - (S0 * du[:, None, :]).sum(-1)
                dv[i], db[i], dg[i] = du, (dn * u).sum(-1), (D0 * S0).sum((-1, -2))
                gsize = torch.maximum(gsize, torch.maximum(D1.norm(dim=-2), D0.norm(dim=-2)))
                D = a * D0
            dh0[r] = D
            bh[r] = self.eps * gsize[:, None, :]
            for i in rows:
                kn, qn = self.k[i].norm(dim=-1), self.q[i].norm(dim=-1)
                both = (gsize * size).sum(-1)
                bq[i] = (abs(self.scale) * (size * do[i].abs()).sum(-1))[:, None]
                bk[i] = 2 * both[:, None]
                bv[i] = self.b[i][:, None] * kn[:, None] * gsize
                bb[i] = 2 * kn * both
                # sums over a chunk of q.dq, k.dk's two parts and the states' product
                bg[i] = 16 * ((2 * kn + 1) * both + qn * bq[i].amax(-1))

        def done(g, b, shared=False):
            if shared:
                g, b = (x.view(n, self.H, G // self.H, -1).sum(2) for x in (g, b))
            return g, U[dtype] * g.abs() + self.eps * b + TINY[dtype]

        return [done(dq, bq, True), done(dk, bk, True), done(dv, bv), done(dg, bg), done(db, bb), (dh0, bh + 1e-37)]


def inputs(n, H, G, dk, dv, dtype, seed=0, keys="random"):
    """q, k, v, decay, beta of n rows.  keys: "random" of length 1, or "alike" (each near the one before, as neighbouring
    samples of a ray are)."""
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn(n, H, dk, generator=g), torch.randn(n, H, dk, generator=g)
    if keys == "alike":
        k = k[:1] + 0.05 * torch.cumsum(k, 0) / max(1.0, n ** 0.5)
    q, k = q / q.norm(dim=-1, keepdim=True), 0.99 * k / k.norm(dim=-1, keepdim=True)
    v = torch.randn(n, G, dv, generator=g)
    decay = -torch.nn.functional.softplus(torch.randn(n, G, generator=g) * 1.5 - 3)
    beta = torch.sigmoid(torch.randn(n, G, generator=g) + (3.0 if keys == "alike" else 0.0))
    return [x.to(dtype) for x in (q, k, v, decay, beta)]
