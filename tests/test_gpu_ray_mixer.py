"""The mixer: norm, delta rule and blended experts together, from the samples to the composited colour and back."""
import pytest
import torch

from delta_oracle import Delta
from ray_oracle import ray_set

pytestmark = pytest.mark.gpu


def _make(lens, width=32, heads=2, dtype=torch.float32, seed=2):
    import ray_model
    torch.manual_seed(seed)
    rays = ray_set(lens)
    n = rays[3]
    samples = torch.rand(n, 4)
    features = torch.randn(n, 10)
    model = ray_model.RayMixer(10, width=width, heads=heads, dtype=dtype)
    for name, p in model.named_parameters():
        if p.dim() == 1 or name in ("b_1", "b_2"):
            torch.nn.init.normal_(p, mean=1.0 if name[0] == "n" else 0.0, std=0.3)
    return model, samples, features, rays


def _cuda(rays):
    import ray_ops
    return ray_ops.RaySet(*(x.cuda() for x in rays[:3]))


def test_blend():
    """Weights of a sample's two regions sum to 1, are even at a face and do not jump across it; outside there is nobody."""
    import ray_model
    m = ray_model.RayMixer(4, cells=3)
    s = torch.tensor([[1 / 3 - 1e-6, 0.5, 0.5, 0], [1 / 3 + 1e-6, 0.5, 0.5, 0], [0.5, 0.5, 0.5, 0], [0.0, 0.5, 0.5, 0],
                      [0.5, 0.5, 0.99, 0], [0.4, 0.5, 0.55, 0]])
    ids, w = m.blend(s)
    assert torch.allclose(w.sum(1), torch.ones(6))
    assert ids.tolist() == [[12, 13], [13, 12], [13, -1], [12, -1], [22, -1], [13, 12]]
    assert torch.allclose(w[:2], torch.full((2, 2), 0.5), atol=1e-5) and torch.equal(w[2:5, 1], torch.zeros(3))
    assert abs(float(w[5, 1]) - 0.3) < 1e-5


def test_matches_plain_operations():
    """Colour and gradients in single precision against the formulas in 64 bits (CPU): rays of several lengths, one empty."""
    model, samples, features, rays = _make([7, 0, 1, 40])
    n = rays[3]
    weight = torch.randn(4, 3)

    class Rule(torch.autograd.Function):  # the oracle's values and gradients
        @staticmethod
        def forward(ctx, *x):
            ctx.d = Delta(*x, rays)
            return ctx.d.o

        @staticmethod
        def backward(ctx, do):
            return tuple(g for g, _ in ctx.d.backward(do, None, torch.float32)[:5])

    def plain(m):
        d = {k: v.detach().double().requires_grad_() for k, v in m.named_parameters()}

        def norm(x, i):
            return torch.nn.functional.layer_norm(x, (32,), d[f"n_{i}"], d[f"m_{i}"], 1e-5)

        x = features.double() @ d["W_in"].T
        h = norm(x, 1)
        q, k, v = (h @ d["W_qkv"].T).view(n, 3, 2, 16).unbind(1)
        q, k = (t / t.norm(dim=-1, keepdim=True) for t in (q, k))
        decay, beta = (h @ d["W_gates"].T + d["b_gates"]).chunk(2, 1)
        o = Rule.apply(q, k, v, -torch.nn.functional.softplus(decay), torch.sigmoid(beta))
        x = x + o.reshape(n, -1) @ d["W_o"].T
        ids, w = m.blend(samples)
        h = norm(x, 2)
        for j in range(2):
            e = ids[:, j].long().clamp(min=0)
            y = torch.relu(torch.matmul(d["W_1"][e], h[:, :, None])[..., 0] + d["b_1"][e])
            y = torch.matmul(d["W_2"][e], y[:, :, None])[..., 0] + d["b_2"][e]
            x = x + torch.where(ids[:, j] >= 0, w[:, j].double(), 0.0)[:, None] * y
        y = norm(x, 3) @ d["W_out"].T + d["b_out"]
        z, c = torch.sigmoid(y[:, :1]), torch.sigmoid(y[:, 1:])
        colours = []
        for r in range(4):
            state = torch.zeros(3, dtype=torch.float64)
            for i in range(int(rays[1][r]) + int(rays[0][r]) - 1, int(rays[1][r]) - 1, -1):
                state = (1 - z[i]) * state + z[i] * c[i]
            colours.append(state)
        colour = torch.stack(colours)
        (colour * weight.double()).sum().backward()
        return colour.detach(), {k: p.grad for k, p in d.items()}

    want, grads = plain(model)
    model = model.cuda()
    colour = model(samples.cuda(), features.cuda(), _cuda(rays))
    (colour * weight.cuda()).sum().backward()
    # some twenty single precision operations in a row, sums of up to 64 terms, each relative to its largest operands
    assert float((colour.detach().cpu().double() - want).abs().max()) < 2.0 ** -15
    for k, p in model.named_parameters():
        off = float((p.grad.cpu().double() - grads[k]).abs().max())
        assert off < 2.0 ** -13 * float(grads[k].abs().max()) + 2.0 ** -20, (k, off)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_by_sample(dtype):
    """Rays looked at sample by sample, with their states: what one look along them gives."""
    R, T = 9, 21
    model, samples, features, _ = _make([T] * R, dtype=dtype)
    model = model.cuda()
    samples, features = samples.cuda(), features.cuda()
    with torch.no_grad():
        whole = model.look(samples, features, _cuda(ray_set([T] * R)))
        state, got = model.states(R), torch.empty_like(whole)
        one = _cuda(ray_set([1] * R))
        for t in range(T):
            rows = torch.arange(R, device="cuda") * T + t
            got[rows] = model.look(samples[rows], features[rows], one, state)
    # the same numbers but for the order of sums; in bfloat16 an o may so round to the next step, 2^-8 of itself, and passes
    # on through two more layers
    bound = 2.0 ** -14 if dtype == torch.float32 else 2.0 ** -4
    assert float((got - whole).abs().max()) < bound * max(1.0, float(whole.abs().max()))


def test_trains():
    """The example runs, and two runs give the same bits."""
    import ray_model
    a = ray_model.train(steps=6, num_rays=256, seed=1, model="mixer")
    b = ray_model.train(steps=6, num_rays=256, seed=1, model="mixer")
    assert len(a) == 6 and a == b and all(v == v for v in a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_rays_miss(dtype):
    """A batch without samples: black rays, gradients of 0."""
    model, samples, features, rays = _make([0, 0, 0], dtype=dtype)
    model = model.cuda()
    colour = model(samples.cuda(), features.cuda(), _cuda(rays))
    assert colour.shape == (3, 3) and not colour.any()
    colour.sum().backward()
    assert all(p.grad is None or not p.grad.any() for p in model.parameters())
