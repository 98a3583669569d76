"""What the bounds of delta_whole accept and what they reject: right values rounded to the type; not zeros, a hundredth more, a
row's shift or a term left out."""
import pytest
import torch

from delta_oracle import Delta
from delta_whole import CASES, make, off, wanted


def _all(case):
    rays, x, h0, do, dlast = made = make(case)
    return rays, wanted(case, rays, x, h0, do, dlast), made


@pytest.mark.parametrize("case", CASES, ids=str)
def test_accepts_and_rejects(case):
    rays, want, (_, x, h0, do, dlast) = _all(case)
    right = {k: v.to(torch.float32 if k in ("last", "dh0") else case[5]) for k, (v, _) in want.items()}
    assert not off(case, rays, right, want)
    # the same gradients as the row by row oracle's
    ref = Delta(*x, rays, h0, reverse=case[7]).backward(do, dlast, case[5])
    for name, (e, _) in zip(("dq", "dk", "dv", "ddecay", "dbeta", "dh0"), ref):
        if name in want:
            assert float((want[name][0] - e).abs().max()) < 1e-12 * (1 + float(e.abs().max())), name
    g = torch.Generator().manual_seed(3)
    for name, t in right.items():
        v = want[name][0]
        every = torch.arange(len(case[0]))
        held = (every if name in ("last", "dh0") else rays[2])[:, None] == every
        norms = v.reshape(*want[name][1].shape, -1).square().sum(-1).T @ held.double()
        some = int((norms > 0).sum())  # rays and heads that have any
        wrong = dict(zeros=torch.zeros_like(v), more=1.01 * v, noise=v + 0.01 * v.square().mean().sqrt() * torch.randn(v.shape, generator=g))
        if name not in ("last", "dh0"):
            wrong["shifted"] = v.roll(1, 0)
        for how, w in wrong.items():
            bad = off(case, rays, {name: w}, want)
            # in every ray and head, but for noise, which is nothing beside a large ray's or head's values
            assert bad and (how == "noise" or len(bad) >= 0.9 * some), (name, how, len(bad), some)


@pytest.mark.parametrize("case", [c for c in CASES if max(c[0]) > 32], ids=str)
def test_rejects_terms_left_out(case):
    """A decay's gradient without the states' product at its chunk's end, and gradients that do not pass a chunk's border."""
    rays, want, (_, x, h0, do, dlast) = _all(case)
    d = Delta(*x, rays, h0, reverse=case[7])
    v = want["ddecay"][0]
    without, cut = v.clone(), {k: want[k][0].clone() for k in ("dk", "dv", "dbeta")}
    r = max(range(len(case[0])), key=lambda i: case[0][i])
    rows = d.rows[r]
    at = (len(rows) - 1) // 16 * 16  # the last chunk's first place, and the chunk before it
    part = (torch.tensor([at]), torch.tensor([0]), torch.zeros(at, dtype=torch.int32), at)
    first = [t[rows[:at]] for t in x]
    e = Delta(*first, part, None if h0 is None else h0[r:r + 1])
    grads = dict(zip(("dq", "dk", "dv", "ddecay", "dbeta"), (t for t, _ in e.backward(do[rows[:at]], None, case[5]))))
    for k in cut:
        cut[k][rows[:at]] = grads[k]
    without[rows[:at]] = grads["ddecay"]
    for name, w in dict(cut, ddecay=without).items():
        assert any(b[1] == r for b in off(case, rays, {name: w}, want)), name
