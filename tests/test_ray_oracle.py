"""The 64-bit oracles of the operators along rays: their gradients against differences of their own values."""
import pytest
import torch

from ray_oracle import Attention, Scan, ray_set, seen_mask

F64 = torch.float64


def _slope(f, x, d, e=1e-6):
    return float(f(x + e * d) - f(x - e * d)) / (2 * e)


@pytest.mark.parametrize("cap,slopes,causal", [(0.0, False, False), (3.0, True, True)])
def test_attention_gradients_against_differences(cap, slopes, causal):
    g = torch.Generator().manual_seed(3)
    rays = ray_set([5, 0, 1, 9], gap=2)
    n = rays[3]
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=F64)  # noqa: E731
    q, k, v, do = rnd(n, 4, 8), rnd(n, 2, 8), rnd(n, 2, 8), rnd(n, 4, 8)
    t = torch.rand(n, generator=g, dtype=F64)
    seen = seen_mask(rays, rays, causal, torch.tensor([2, 0, 0, 3]) if causal else None)
    opt = dict(scale=0.3, cap=cap, slopes=torch.tensor([1.0, .5, .25, .1]) if slopes else None, t_q=t, t_k=t)
    f = lambda q, k, v: (Attention(q, k, v, seen, **opt).o * do).sum()  # noqa: E731
    grads = [x for x, _ in Attention(q, k, v, seen, **opt).backward(do, torch.float32)]
    for i, x in enumerate((q, k, v)):
        d = rnd(*x.shape)
        at = lambda y: f(*[y if j == i else z for j, z in enumerate((q, k, v))])  # noqa: B023,E731
        assert abs(_slope(at, x, d) - float((grads[i] * d).sum())) < 1e-7


@pytest.mark.parametrize("reverse", [False, True])
def test_scan_gradients_against_differences(reverse):
    g = torch.Generator().manual_seed(4)
    rays = ray_set([7, 0, 1, 12], gap=1)
    n = rays[3]
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=F64)  # noqa: E731
    gate, x, dh, h0, dlast = rnd(n, 3), rnd(n, 3), rnd(n, 3), rnd(4, 3), rnd(4, 3)

    def f(gate, x, h0):
        s = Scan(gate, x, rays, h0, reverse)
        return (s.h * dh).sum() + (s.last * dlast).sum()

    grads = [y for y, _ in Scan(gate, x, rays, h0, reverse).backward(dh, dlast, torch.float32)]
    for i, y in enumerate((gate, x, h0)):
        d = rnd(*y.shape)
        at = lambda w: f(*[w if j == i else z for j, z in enumerate((gate, x, h0))])  # noqa: B023,E731
        assert abs(_slope(at, y, d) - float((grads[i] * d).sum())) < 1e-7
