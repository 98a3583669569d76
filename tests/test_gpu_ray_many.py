"""Calls of more threads than one axis of a launch can count (2^32): the last rows and rays have their results too."""
import pytest
import torch

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def _room(request):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 120 << 30:
        pytest.skip("needs 120 GiB of the card's memory")
    yield
    torch.cuda.empty_cache()


def _even(n, rays, per):
    """`rays` rays of `per` rows each, the last one shorter if n ends before."""
    import ray_ops
    counts = torch.full((rays,), per, **I32)
    counts[-1] = n - (rays - 1) * per
    offsets = torch.arange(rays, **I32) * per
    ids = torch.arange(rays, **I32).view(-1, 1).expand(-1, per).reshape(-1)[:n]
    return ray_ops.RaySet(counts, offsets, ids)


def _fill(x, seed=0):
    """Small values that repeat every 4096 rows, so that rows far apart can be compared."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    one = torch.randn(4096, *x.shape[1:], generator=g, device="cuda").to(x.dtype)
    for i in range(0, x.shape[0], 4096):
        x[i:i + 4096] = one[:x.shape[0] - i]
    return x


def test_attention_of_many_heads():
    """2^24 + 1024 blocks of 64 rows of a head, forward and backward: the last rays as the first ones, bit for bit."""
    import ray_ops
    n, heads = (1 << 20) + 64, 1024
    rays = _even(n, n // 64, 64)
    q = _fill(torch.empty(n, heads, 8, dtype=torch.bfloat16, device="cuda"))
    k, v = (_fill(torch.empty(n, 1, 8, dtype=torch.bfloat16, device="cuda"), s) for s in (1, 2))
    o, lse = ray_ops.ray_attention(q, k, v, rays, causal=True)
    dq, dk, dv = ray_ops.ray_attention_backward(q, q, k, v, o, lse, rays, causal=True)
    for x in (o, lse, dq, dk, dv):
        for i in (n - 64, n // 2 - n // 2 % 4096):
            assert torch.equal(x[i:i + 64], x[:64])
        assert torch.isfinite(x[-64:].float()).all() and x[-64:].any()


def test_a_query_at_a_time_of_many_rays():
    """2^26 + 4 rays of six keys and a query."""
    import ray_ops
    rays, heads = (1 << 26) + 4, 16
    keys = _even(rays * 6, rays, 6)
    each = torch.arange(rays, **I32)
    queries = ray_ops.RaySet(torch.ones(rays, **I32), each, each)
    q = torch.empty(rays, heads, 8, dtype=torch.bfloat16, device="cuda")
    q[:] = torch.randn(heads, 8, device="cuda").to(q.dtype)
    k, v = (torch.empty(rays, 6, 8, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k[:], v[:] = (torch.randn(6, 8, device="cuda").to(k.dtype) for _ in range(2))
    o, lse = ray_ops.ray_attention(q, k.view(-1, 1, 8), v.view(-1, 1, 8), queries, keys)
    for x in (o, lse):
        assert x[0].any() and torch.isfinite(x[0].float()).all()
        for i in range(0, rays, 1 << 22):
            assert torch.equal(x[i:i + (1 << 22)], x[:1].expand_as(x[i:i + (1 << 22)]))


@pytest.mark.parametrize("C,dtype", [(512, torch.bfloat16), (257, torch.float32)])
def test_recurrence_of_many_rays(C, dtype):
    """2^24 + 300 rays, all but the last without rows: their states are what they start from."""
    import ray_ops
    R = (1 << 24) + 300
    counts, zero = torch.zeros(R, **I32), torch.zeros(R, **I32)
    counts[-1] = 2
    rays = ray_ops.RaySet(counts, zero, torch.full((2,), R - 1, **I32))
    h0 = torch.ones(R, C, device="cuda")
    gate, x = torch.zeros(2, C, dtype=dtype, device="cuda"), torch.full((2, C), 3.0, dtype=dtype, device="cuda")
    h, last, marks = ray_ops.ray_scan(gate, x, rays, h0=h0, marks=True)
    assert (h[0] == 2.0).all() and (h[1] == 2.5).all()
    assert (last[-1] == 2.5).all() and (last[:-1] == 1.0).all()
    dgate, dx, dh0 = ray_ops.ray_scan_backward(torch.zeros_like(x), gate, x, marks, rays, dlast=h0, h0=h0)
    assert (dx[1] == 0.5).all() and (dx[0] == 0.25).all() and (dh0[-1] == 0.25).all() and (dh0[:-1] == 1.0).all()


def test_experts_of_many_rows():
    """The largest number of rows: 2^24 tiles of slots and the last ones of each expert."""
    import ray_ops
    n, E = 0x7FFFFF00, 8
    ids = torch.empty(n, **I32)
    for i in range(0, n, 1 << 28):
        ids[i:i + (1 << 28)] = torch.arange(i, min(n, i + (1 << 28)), **I32) % 4096 % E
    x = torch.empty(n, 8, dtype=torch.bfloat16, device="cuda")
    x.view(-1, 256, 8)[:] = torch.randn(256, 8, device="cuda").to(x.dtype)
    W = torch.randn(E, 8, 8, device="cuda").to(x.dtype)
    plan = ray_ops.expert_plan(ids, E)
    y = ray_ops.expert_linear(x, W, None, plan)
    Ws, xs = W[ids[:256].long()].double(), x[:256].double()[:, :, None]
    want, size = torch.matmul(Ws, xs)[..., 0], torch.matmul(Ws.abs(), xs.abs())[..., 0]
    # eight products and sums in single precision, one rounding to the type
    assert ((y[:256].double() - want).abs() <= 2.0 ** -8 * want.abs() + 16 * 2.0 ** -24 * size).all()
    for i in range(0, n, 1 << 26):
        part = y[i:i + (1 << 26)].view(-1, 256, 8)
        assert torch.equal(part, y[:256].expand_as(part))
