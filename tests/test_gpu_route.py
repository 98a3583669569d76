"""Rows to several experts and back against their definition, place by place, in 64 bits.

Bounds: u = eps / 2 of a type; sums of k weighted rows have k products and k sums in float, dot products over a width of w
are taken by lanes of at most 8 w / 64 + 8 terms and by halves after that."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def make(n, k, experts, width, dtype, seed=0, dropped=0.2):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (n, k), generator=g, dtype=torch.int32)  # the same expert twice is allowed
    lost = torch.rand(n, k, generator=g) < dropped
    ids = torch.where(lost, torch.tensor([-1, experts, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)[
        torch.randint(0, 4, (n, k), generator=g)], ids)
    x = torch.randn(n, width, generator=g).to(dtype)
    y = torch.randn(n * k, width, generator=g).to(dtype)
    w = torch.rand(n, k, generator=g)
    return ids.cuda(), x.cuda(), y.cuda(), w.cuda()


def slots_of(ids, experts):
    """Slot of each place, and whether it has an expert: places in the order of (expert, place)."""
    flat = ids.cpu().long().view(-1)
    inside = (flat >= 0) & (flat < experts)
    order = sorted(range(len(flat)), key=lambda p: (int(flat[p]) if inside[p] else experts, p))
    slots = torch.empty(len(flat), dtype=torch.long)
    slots[torch.tensor(order, dtype=torch.long)] = torch.arange(len(flat))
    return slots.view(ids.shape), inside.view(ids.shape)


def check(ids, experts, x, y, w, dout, dxs):
    import ray_ops
    n, k = ids.shape
    width, u = x.shape[1], torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal
    route = ray_ops.expert_route(ids, experts)
    slots, inside = slots_of(ids, experts)
    assert torch.equal(route.slots.cpu().long(), slots)
    xs = ray_ops.expert_dispatch(x, route)
    X, Y, D, DXS = (t.cpu().double() for t in (x, y, dout, dxs))
    W = torch.ones(n, k, dtype=torch.float64) if w is None else w.cpu().double()
    want = torch.zeros(n * k, width, dtype=torch.float64)
    want[slots[inside]] = X[torch.nonzero(inside)[:, 0]]
    assert torch.equal(xs.cpu().double(), want)
    total = ray_ops.expert_combine(y, route, w)
    Yk = torch.where(inside[:, :, None], Y[slots], 0.0)
    Wk = torch.where(inside, W, 0.0)
    E = (Wk[:, :, None] * Yk).sum(1)
    size = (Wk[:, :, None] * Yk).abs().sum(1)
    assert ((total.cpu().double() - E).abs() <= u * E.abs() + 2 * k * U32 * size + tiny).all()
    dy, dw = ray_ops.expert_combine_backward(dout, y, route, w)
    want = torch.zeros(n * k, width, dtype=torch.float64)
    want[slots[inside]] = (Wk[:, :, None] * D[:, None, :])[inside]
    assert ((dy.cpu().double() - want).abs() <= (u + 2 * U32) * want.abs() + tiny).all()
    E = (D[:, None, :] * Yk).sum(2)
    size = (D[:, None, :] * Yk).abs().sum(2)
    assert ((dw.cpu().double() - E).abs() <= (width / 8 + 32) * U32 * size).all()
    assert not dw[~inside.cuda()].any() and not dy[slots[~inside].cuda()].any()
    dx = ray_ops.expert_dispatch_backward(dxs, route)
    G = torch.where(inside[:, :, None], DXS[slots], 0.0)
    assert ((dx.cpu().double() - G.sum(1)).abs() <= u * G.sum(1).abs() + 2 * k * U32 * G.abs().sum(1) + tiny).all()
    return route


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 7, 8, 24, 64, 72, 512, 520, 1000, 1024])
def test_widths(width, dtype):
    ids, x, y, w = make(37, 3, 5, width, dtype, seed=width)
    check(ids, 5, x, y, w, x.flip(0), y.flip(0))


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 8, 13])
@pytest.mark.parametrize("experts", [1, 6, 200])
def test_places(k, experts):
    ids, x, y, w = make(61, k, experts, 16, torch.bfloat16, seed=k)
    check(ids, experts, x, y, w, x.flip(0), y.flip(0))
    check(ids, experts, x, y, None, x.flip(0), y.flip(0))


@pytest.mark.parametrize("n", [1, 2, 5000])
def test_rows(n):
    ids, x, y, w = make(n, 2, 9, 40, torch.float16, seed=n)
    check(ids, 9, x, y, w, x.flip(0), y.flip(0))


def test_nobody():
    """Every place without an expert, and no rows at all."""
    import ray_ops
    ids, x, y, w = make(20, 2, 4, 24, torch.float32)
    check(torch.full_like(ids, -1), 4, x, y, w, x, y)
    route = ray_ops.expert_route(torch.empty(0, 3, dtype=torch.int32, device="cuda"), 4)
    e = torch.empty(0, 24, device="cuda")
    assert ray_ops.expert_dispatch(e, route).shape == ray_ops.expert_combine(e, route).shape == (0, 24)
    dy, dw = ray_ops.expert_combine_backward(e, e, route, torch.empty(0, 3, device="cuda"))
    assert dy.shape == (0, 24) and dw.shape == (0, 3)


def test_sick_slots_of_no_expert():
    """What y, weights and gradients hold at places of no expert reaches nothing."""
    import ray_ops
    ids, x, y, w = make(300, 2, 4, 24, torch.bfloat16)
    slots, inside = slots_of(ids, 4)
    route = ray_ops.expert_route(ids, 4)
    sick_y, sick_w = y.clone(), w.clone()
    sick_y[slots[~inside].cuda()] = float("nan")
    sick_w[~inside.cuda()] = float("inf")
    assert torch.equal(ray_ops.expert_combine(y, route, w), ray_ops.expert_combine(sick_y, route, sick_w))
    for p, q in zip(ray_ops.expert_combine_backward(x, y, route, w), ray_ops.expert_combine_backward(x, sick_y, route, sick_w)):
        assert torch.equal(p, q)
    assert torch.equal(ray_ops.expert_dispatch_backward(y, route), ray_ops.expert_dispatch_backward(sick_y, route))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    """Rows inside wider ones, at any start, and one row for all."""
    ids, x, y, w = make(40, 2, 4, 64, dtype)

    def inside_of(t, shift, pad):
        wide = torch.full((t.shape[0], 64 + shift + pad), float("nan"), dtype=dtype, device="cuda")
        wide[:, shift:shift + 64] = t
        return wide[:, shift:shift + 64]

    for shift, pad in ((0, 8), (8, 16), (1, 2)):
        check(ids, 4, inside_of(x, shift, pad), inside_of(y, shift, pad), w, inside_of(x.flip(0), shift, pad),
              inside_of(y.flip(0), shift, pad))
    check(ids, 4, x[:1].expand(40, 64), y[:1].expand(80, 64), w, x[:1].expand(40, 64), y[:1].expand(80, 64))


def test_layers_in_slot_order():
    """Dispatch, two layers of experts in slot order, weighted sum: against the layers of each place, forward and backward."""
    import ray_ops
    g = torch.Generator().manual_seed(4)
    n, k, E, d = 50, 3, 4, 16
    ids, x, _, w = make(n, k, E, d, torch.float32, dropped=0.1)
    W1, W2 = (torch.randn(E, d, d, generator=g).cuda() / 4 for _ in range(2))
    b1 = torch.randn(E, d, generator=g).cuda()
    leaves = [t.requires_grad_() for t in (x, w, W1, b1, W2)]
    route = ray_ops.expert_route(ids, E)
    h = ray_ops.ExpertDispatch.apply(x, route)
    h = ray_ops.ExpertLinear.apply(h, W1, b1, route.plan, True, True, True)
    h = ray_ops.ExpertLinear.apply(h, W2, None, route.plan, False, True, True)
    out = ray_ops.ExpertCombine.apply(h, route, w)
    dout = torch.randn(n, d, generator=g).cuda()
    got = torch.autograd.grad(out, leaves, dout)
    ref = [t.detach().cpu().double().requires_grad_() for t in leaves]
    X, Wt, A, B, C = ref
    inside = (ids >= 0) & (ids < E)
    total = torch.zeros(n, d, dtype=torch.float64)
    for i in range(n):
        for j in range(k):
            if inside[i, j]:
                e = int(ids[i, j])
                total = total.index_add(0, torch.tensor([i]), (Wt[i, j] * (C[e] @ torch.relu(A[e] @ X[i] + B[e])))[None])
    want = torch.autograd.grad(total, ref, dout.cpu().double())
    # three products of 16 terms in float, each within 20 of its steps
    assert float((out.detach().cpu().double() - total.detach()).abs().max()) < 64 * U32 * float(total.abs().max()) * 4
    for p, q in zip(got, want):
        assert float((p.cpu().double() - q).abs().max()) < 512 * U32 * max(1.0, float(q.abs().max()))


def test_autograd_once():
    import ray_ops
    ids, x, y, w = make(10, 2, 4, 8, torch.float32)
    route = ray_ops.expert_route(ids, 4)
    y.requires_grad_(), w.requires_grad_(), x.requires_grad_()
    for out, t in ((ray_ops.ExpertCombine.apply(y, route, w), w), (ray_ops.ExpertCombine.apply(y, route, w), y),
                   (ray_ops.ExpertDispatch.apply(x, route), x)):
        grad, = torch.autograd.grad((out ** 2).sum(), [t], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated once"):
            (grad ** 2).sum().backward()


def test_graph_replays():
    """Route and sums captured, replayed with other ids and rows: the eager bits each time."""
    import ray_ops
    n, k, E, d = 9001, 2, 7, 64

    def both(ids, x, y, w):
        route = ray_ops.expert_route(ids, E)
        return (route.slots, ray_ops.expert_dispatch(x, route), ray_ops.expert_combine(y, route, w),
                *ray_ops.expert_combine_backward(x, y, route, w))

    held = [t.clone() for t in make(n, k, E, d, torch.bfloat16)]
    both(*held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(*held)
    for seed in (1, 2, 3):
        new = make(n, k, E, d, torch.bfloat16, seed=seed)
        for h, t in zip(held, new):
            h.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, both(*new)))


def test_slots_past_32_bit_offsets():
    """Slots more than 2^32 bytes apart."""
    import ray_ops
    n, k, width = 9000, 8, 32768
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    ids = (torch.arange(n * k, device="cuda", dtype=torch.int32) % 3).view(n, k)
    route = ray_ops.expert_route(ids, 3)
    x = torch.arange(n, device="cuda").remainder(251).to(torch.bfloat16)[:, None].expand(n, width).contiguous()
    xs = ray_ops.expert_dispatch(x, route)
    assert xs.numel() * 2 > 1 << 32
    back = ray_ops.expert_dispatch_backward(xs, route)  # k times the row, whole numbers below 2^11
    assert torch.equal(back[:, 5].float(), (x[:, 5].float() * k).to(torch.bfloat16).float())
    assert torch.equal(back[:, -1], back[:, 0])
