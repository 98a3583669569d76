"""Attention with many heads on one key head, in the form that its sizes take."""
import pytest
import torch

from ray_oracle import Attention, close, ray_set, seen_mask

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ty", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G", [(17, 1), (40, 1), (64, 2)])
@pytest.mark.parametrize("nq,nk", [([90, 3, 41], None), ([1, 2, 1], [700, 30, 300]), ([20, 9, 1], [90, 64, 500])])
def test_many_heads_on_a_key_head(ty, H, G, nq, nk):
    import ray_ops
    qs = ray_set(nq)
    ks = qs if nk is None else ray_set(nk, gap=1)
    g = torch.Generator().manual_seed(61)
    rnd = lambda n, h: torch.randn(n, h, 24, generator=g).to(ty)  # noqa: E731
    q, k, v, do = rnd(qs[3], H), rnd(ks[3], G), rnd(ks[3], G), rnd(qs[3], H)
    ref = Attention(q, k, v, seen_mask(qs, ks, True, None), scale=24 ** -0.5, cap=5.0)
    rq, rk = (ray_ops.RaySet(*(x.cuda() for x in s[:3])) for s in (qs, ks))
    a = [x.cuda() for x in (q, k, v)]
    o, lse = ray_ops.ray_attention(*a, rq, rk, causal=True, cap=5.0)
    close(o, ref.o, ref.o_bound(ty), "o")
    close(lse, ref.lse, ref.lse_bound(), "lse")
    got = ray_ops.ray_attention_backward(do.cuda(), *a, o, lse, rq, rk, causal=True, cap=5.0)
    for x, (want, bound), name in zip(got, ref.backward(do, ty), ("dq", "dk", "dv")):
        close(x, want, bound, name)
