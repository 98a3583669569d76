"""Prefixes at and past their ends: b < prefix shows no key where the prefix is negative, and all where it is large."""
import pytest
import torch

from ray_oracle import Attention, close, ray_set, seen_mask

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
PREFIX = [-1, -2 ** 31, 3, 0, 2 ** 31 - 1]


@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("nq,nk", [([20, 40, 9, 5, 30], None), ([2, 1, 3, 1, 2], [70, 900, 8, 33, 300]),
                                   ([30, 9, 4, 2, 1], [5, 2, 4, 1, 0])])
def test_prefix_of_any_value(ty, nq, nk):
    """All rows among themselves, few queries over long rays, and more queries than keys."""
    import ray_ops
    qs = ray_set(nq, gap=1)
    ks = qs if nk is None else ray_set(nk, gap=2)
    prefix = torch.tensor(PREFIX, dtype=torch.int32)
    g = torch.Generator().manual_seed(51)
    rnd = lambda n, h: torch.randn(n, h, 32, generator=g).to(TYPES[ty])  # noqa: E731
    q, k, v, do = rnd(qs[3], 4), rnd(ks[3], 2), rnd(ks[3], 2), rnd(qs[3], 4)
    ref = Attention(q, k, v, seen_mask(qs, ks, True, prefix), scale=32 ** -0.5)
    rq, rk = (ray_ops.RaySet(*(x.cuda() for x in s[:3])) for s in (qs, ks))
    a = [x.cuda() for x in (q, k, v)]
    o, lse = ray_ops.ray_attention(*a, rq, rk, causal=True, prefix=prefix.cuda())
    close(o, ref.o, ref.o_bound(q.dtype), "o")
    close(lse, ref.lse, ref.lse_bound(), "lse")
    got = ray_ops.ray_attention_backward(do.cuda(), *a, o, lse, rq, rk, causal=True, prefix=prefix.cuda())
    for x, (want, bound), name in zip(got, ref.backward(do, q.dtype), ("dq", "dk", "dv")):
        close(x, want, bound, name)


def test_prefix_of_uint32():
    """Values past 2^31 of an unsigned prefix are large, not negative."""
    import ray_ops
    rays = ray_ops.RaySet(*(x.cuda() for x in ray_set([20, 9])[:3]))
    x = torch.randn(29, 2, 16, device="cuda")
    large = torch.tensor([2 ** 32 - 1, 2 ** 31], dtype=torch.uint32).cuda()
    o, lse = ray_ops.ray_attention(x, x, x, rays, causal=True, prefix=large)
    all_o, all_lse = ray_ops.ray_attention(x, x, x, rays)
    assert torch.equal(o, all_o) and torch.equal(lse, all_lse)
