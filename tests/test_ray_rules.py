"""Which form of attention a call takes, seen by the scratch it asks for (a query at a time, split over the keys, needs
some; whole tiles of queries need none in the forward pass).  Nothing here reaches the GPU."""
import ctypes as C

import pytest

import ffn_lib as fl


def _scratch(rays, n_q, n_k, heads, kv_heads, dim=64, dtype=2):
    a = fl.FfnRayAttn(dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, scale=0.1, q_rays=fl.FfnRaySet(num_rays=rays, n=n_q),
                      k_rays=fl.FfnRaySet(num_rays=rays, n=n_k))
    n = C.c_uint64()
    assert fl.load().ffn_ray_attention_workspace(C.byref(a), 0, C.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("rays,rows,heads", [(2, 3000, 64), (2, 3000, 128), (1, 2000, 32), (1, 1500, 256)])
def test_many_heads_on_one_key_head_take_tiles(rays, rows, heads):
    """A query at a time reads its keys once for every 16 heads that share them; tiles of queries are the faster then."""
    assert _scratch(rays, rows, rows, heads, 1) == 0


@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (8, 2), (32, 1), (64, 1)])
def test_few_queries_over_long_rays_take_a_query_at_a_time(heads, kv_heads):
    assert _scratch(64, 64, 64 * 16384, heads, kv_heads) > 0


@pytest.mark.parametrize("rays,n_q,keys,heads,kv_heads", [(64, 1024, 8192, 64, 1), (64, 1024, 8192, 8, 2)])
def test_a_query_at_a_time_lasts_longer_in_the_backward(rays, n_q, keys, heads, kv_heads):
    """Where tiles take as long forward, their backward takes longer.  (Scratch beyond the products D, 4 bytes a row.)"""
    a = fl.FfnRayAttn(dtype=2, heads=heads, kv_heads=kv_heads, dim=64, scale=0.1, q_rays=fl.FfnRaySet(num_rays=rays, n=n_q),
                      k_rays=fl.FfnRaySet(num_rays=rays, n=rays * keys))
    n = C.c_uint64()
    assert fl.load().ffn_ray_attention_workspace(C.byref(a), 1, C.byref(n)) == 0
    assert n.value > 4 * n_q * heads
