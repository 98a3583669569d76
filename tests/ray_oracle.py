"""Plain restatements in 64 bits (CPU) of the operators along rays and of the expert layers, with bounds of the kernels'
rounding: each oracle returns values and, for every value, the sum of magnitudes that its roundings scale with."""
from __future__ import annotations

import math

import torch

F64 = torch.float64
# largest relative error of one rounding to the type
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}


def ray_set(lens, gap=0, shuffle=None):
    """(counts, offsets, ray_ids, n): rays one after the other with `gap` rows of no ray after each."""
    counts = torch.tensor(lens, dtype=torch.int32)
    step = counts + gap
    offsets = (torch.cumsum(step, 0) - step).to(torch.int32)
    n = int(step.sum())
    ids = torch.full((n,), len(lens) + 7, dtype=torch.int32)
    for r, (o, c) in enumerate(zip(offsets.tolist(), counts.tolist())):
        ids[o:o + c] = r
    return counts, offsets, ids, n


def seen_mask(qs, ks, causal, prefix):
    """[n_q, n_k]: what each query row sees, straight from the definition."""
    (qc, qo, _, qn), (kc, ko, _, kn) = qs, ks
    m = torch.zeros(qn, kn, dtype=torch.bool)
    for r in range(len(qc)):
        nq, nk, q0, k0 = int(qc[r]), int(kc[r]), int(qo[r]), int(ko[r])
        a, b = torch.arange(nq)[:, None], torch.arange(nk)[None, :]
        see = torch.ones(nq, nk, dtype=torch.bool)
        if causal:
            see = b <= a + nk - nq
            if prefix is not None:
                see = see | (b < int(prefix[r]))
        m[q0:q0 + nq, k0:k0 + nk] = see
    return m


class Attention:
    """Dense attention over all rows with a mask; rows that see nothing give 0 and -inf."""

    def __init__(self, q, k, v, seen, *, scale, cap=0.0, slopes=None, t_q=None, t_k=None):
        self.H, self.G = q.shape[1], k.shape[1]
        self.q, self.k, self.v = (x.to(F64).transpose(0, 1) for x in (q, k, v))  # [heads, n, dim]
        self.share = torch.arange(self.H) // (self.H // self.G)
        # what is not seen must not matter: NaN and infinities of rows that nobody sees are taken out here
        self.k, self.v = (torch.where(seen.any(0)[None, :, None], x, 0.0) for x in (self.k, self.v))
        self.q = torch.where(seen.any(1)[None, :, None], self.q, 0.0)
        kk, vv = self.k[self.share], self.v[self.share]
        s = scale * (self.q @ kk.transpose(1, 2))
        self.smax = scale * float((self.q.abs() @ kk.abs().transpose(1, 2)).max()) if s.numel() else 0.0
        self.th = torch.tanh(s / cap) if cap > 0 else None
        c = cap * self.th if cap > 0 else s
        if slopes is not None:
            far = (t_q.to(F64)[:, None] - t_k.to(F64)[None, :]).abs()
            c = c - slopes.to(F64)[:, None, None] * far
            self.smax += float(slopes.max()) * float(t_q.abs().max() + t_k.abs().max())
        self.smax += cap
        logits = torch.where(seen, c, -math.inf)
        top = logits.amax(-1, keepdim=True) if s.shape[-1] else torch.full((*s.shape[:2], 1), -math.inf, dtype=F64)
        top = torch.where(top == -math.inf, 0.0, top)
        e = torch.exp(logits - top)
        l = e.sum(-1, keepdim=True)
        self.P = torch.where(l > 0, e / l, 0.0)
        self.lse = (top + torch.log(l))[..., 0].transpose(0, 1)
        self.o_h = self.P @ vv
        self.o = self.o_h.transpose(0, 1)
        self.o_mag = (self.P @ vv.abs()).transpose(0, 1)
        self.scale, self.cap, self.seen = scale, cap, seen
        self.dim = q.shape[2]
        # error of a logit in single precision, and so the relative error of a weight
        self.eps = 2.0 ** -24 * (self.dim + 16) * (self.smax + 1.0)

    def shared(self, x):  # [H, n, d] -> [n, G, d], summed over the query heads of a key head
        return x.view(self.G, self.H // self.G, *x.shape[1:]).sum(1).transpose(0, 1)

    def backward(self, do, dtype):
        """dq, dk, dv and their bounds: a rounding of every weight to the type, of the result, and of o in D = do.o."""
        do = torch.where(self.seen.any(1)[None, :, None], do.to(F64).transpose(0, 1), 0.0)
        kk, vv = self.k[self.share], self.v[self.share]
        D = (do * self.o_h).sum(-1, keepdim=True)
        dl = self.P * (do @ vv.transpose(1, 2) - D)
        if self.cap > 0:
            dl = dl * (1 - self.th ** 2)
        dl = dl * self.scale
        dq, dk, dv = dl @ kk, dl.transpose(1, 2) @ self.q, self.P.transpose(1, 2) @ do
        u, e = U[dtype], 4 * self.eps + 2.0 ** -20
        w = u if dtype != torch.float32 else 0.0
        # weight magnitudes whose relative errors are w (rounding) and e (single precision, before the difference)
        Dmag = (do.abs() * self.o_h.abs()).sum(-1, keepdim=True)
        pmag = self.P * (do.abs() @ vv.abs().transpose(1, 2) + Dmag) * self.scale
        err = w * dl.abs() + e * pmag + w * self.P * Dmag * self.scale
        verr = (w + e) * self.P
        bq = err @ kk.abs() + u * dq.abs()
        bk = err.transpose(1, 2) @ self.q.abs()
        bv = verr.transpose(1, 2) @ do.abs()
        dk, dv, bk, bv = (self.shared(x) for x in (dk, dv, bk, bv))
        t = TINY[dtype]
        return ((dq.transpose(0, 1), 1.1 * bq.transpose(0, 1) + t), (dk, 1.1 * (bk + u * dk.abs()) + t),
                (dv, 1.1 * (bv + u * dv.abs()) + t))

    def o_bound(self, dtype):
        u = U[dtype]
        w = u if dtype != torch.float32 else 0.0
        return 1.1 * (u * self.o.abs() + (w + 4 * self.eps + 2.0 ** -20) * self.o_mag) + TINY[dtype]

    def lse_bound(self):
        return 2 * self.eps + 2.0 ** -20 * (1 + self.lse.abs())


class Scan:
    """The recurrence step by step, and its gradients."""

    def __init__(self, gate, x, rays, h0, reverse):
        counts, offsets, _, n = rays
        C = x.shape[1]
        gate, x = gate.to(F64), x.to(F64)
        self.h, self.mag = torch.zeros(n, C, dtype=F64), torch.zeros(n, C, dtype=F64)
        self.last = torch.zeros(len(counts), C, dtype=F64) if h0 is None else h0.to(F64).clone()
        self.last_mag = self.last.abs()
        self.before = torch.zeros(n, C, dtype=F64)
        self.rows = []
        for r in range(len(counts)):
            o, m = int(offsets[r]), int(counts[r])
            rows = list(range(o, o + m))[::-1] if reverse else list(range(o, o + m))
            self.rows.append(rows)
            s, g = self.last[r].clone(), self.last_mag[r].clone()
            for i in rows:
                z = torch.sigmoid(gate[i])
                self.before[i] = s
                s = (1 - z) * s + z * x[i]
                g = (1 - z) * g + z * x[i].abs()
                self.h[i], self.mag[i] = s, g
            self.last[r], self.last_mag[r] = s, g
        self.gate, self.x = gate, x
        # single precision: a few roundings a step of a state that forgets (its errors decay as it does), and of z
        self.steps = max([1] + [len(r) for r in self.rows])
        self.eps = 2.0 ** -24 * 8 * min(self.steps, 64)

    def backward(self, dh, dlast, dtype):
        n, C = self.x.shape
        dgate, dx = torch.zeros(n, C, dtype=F64), torch.zeros(n, C, dtype=F64)
        bg, bx = torch.zeros(n, C, dtype=F64), torch.zeros(n, C, dtype=F64)
        dh0 = torch.zeros(len(self.rows), C, dtype=F64) if dlast is None else dlast.to(F64).clone()
        d0mag = dh0.abs()
        dh = dh.to(F64)
        u = U[dtype]
        for r, rows in enumerate(self.rows):
            d, g = dh0[r].clone(), d0mag[r].clone()
            for i in reversed(rows):
                z = torch.sigmoid(self.gate[i])
                d = d + dh[i]
                g = g + dh[i].abs()
                dx[i] = z * d
                dgate[i] = d * (self.x[i] - self.before[i]) * z * (1 - z)
                bx[i] = u * dx[i].abs() + self.eps * z * g
                near = self.x[i].abs() + self.before[i].abs() + self.mag[i]
                bg[i] = u * dgate[i].abs() + 2 * self.eps * g * near * z
                d, g = (1 - z) * d, (1 - z) * g
            dh0[r], d0mag[r] = d, g
        t = TINY[dtype]
        return (dgate, 1.1 * bg + t), (dx, 1.1 * bx + t), (dh0, 1.1 * self.eps * d0mag + t)

    def h_bound(self, dtype):
        return 1.1 * (U[dtype] * self.h.abs() + self.eps * self.mag) + TINY[dtype]


def close(got, want, bound, what):
    """Every value within its bound; infinities and NaN equal."""
    got, want = got.detach().cpu().to(F64), want.to(F64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(fine, ((got - want).abs() > bound) | ~torch.isfinite(got), ~same)
    if off.any():
        i = int(off.reshape(-1).nonzero()[0])
        b = bound.expand(want.shape).reshape(-1)[i] if isinstance(bound, torch.Tensor) else bound
        raise AssertionError(f"{what}: {int(off.sum())} of {off.numel()} values off, first at {i}: "
                             f"{float(got.reshape(-1)[i])} for {float(want.reshape(-1)[i])}, bound {float(b)}")
