"""The delta rule as a function of torch keeps states for a backward pass where there may be one, and only there."""
import pytest
import torch

from delta_oracle import Delta, inputs
from ray_oracle import close, ray_set

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[1] * 30, [40, 0, 25]])
def test_marks(lens, monkeypatch):
    import ray_ops
    rays = ray_set(lens)
    set_ = ray_ops.RaySet(*(t.cuda() for t in rays[:3]))
    x = [t.cuda() for t in inputs(rays[3], 1, 2, 16, 24, torch.float32, seed=3)]
    h0 = torch.randn(len(lens), 2, 16, 24, device="cuda")
    made, plain = [], ray_ops.ray_delta
    monkeypatch.setattr(ray_ops, "ray_delta", lambda *a, **k: made.append(k["marks"]) or plain(*a, **k))
    f = ray_ops.RayDelta.apply
    leaf = [t.clone().requires_grad_() for t in x]
    state = h0.clone().requires_grad_()
    with torch.no_grad():
        first = f(*leaf, set_, state)
    second = f(*x, set_, h0)
    with torch.inference_mode():
        f(*x, set_)
    assert made == [False] * 3 and not first[0].requires_grad and not second[0].requires_grad
    # what one call without marks gives
    o, last, _ = plain(*x, set_, h0=h0, last=True)
    for got in (first, second):
        assert torch.equal(got[0], o) and torch.equal(got[1], last)
    want = Delta(*(t.cpu() for t in x), rays, h0.cpu())
    for (e, b), got in zip(zip((want.o, want.last), want.bounds(torch.float32)), second):
        close(got, e, b, "without marks")
    # a gradient of one input alone is enough
    for i in range(6):
        del made[:]
        y = [t.clone().requires_grad_(j == i) for j, t in enumerate((*x, h0))]
        g, = torch.autograd.grad(f(*y[:5], set_, y[5])[0].sum(), [y[i]])
        assert made == [True] and g.shape == y[i].shape and bool(g.abs().sum() > 0)


def test_model_without_gradients():
    """A model that is only asked takes no memory for a backward pass."""
    import ray_ops
    from test_gpu_ray_mixer import _cuda, _make
    model, samples, features, rays = _make([64] * 512, width=64, heads=1)
    model, samples, features, set_ = model.cuda(), samples.cuda(), features.cuda(), _cuda(rays)
    marks = 512 * 2 * 64 * 64 * 4  # a state of a ray every 32 rows
    q = torch.zeros(rays[3], 1, 64, device="cuda")
    gates = torch.zeros(rays[3], 1, device="cuda", requires_grad=True)
    with torch.no_grad():
        for fn in (lambda: ray_ops.RayDelta.apply(q, q, q, gates, gates, set_, None, dict(last=False)),):
            fn()
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            held = torch.cuda.memory_allocated()
            fn()
            assert torch.cuda.max_memory_allocated() - held < marks
        colour = model(samples, features, set_)
    with_grads = model(samples, features, set_)
    # the same kernel, without marks
    assert torch.equal(colour, with_grads.detach())
