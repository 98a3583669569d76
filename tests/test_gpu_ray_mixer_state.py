"""The mixer's gradients where it is asked with the rays' states in hand."""
import pytest
import torch

from ray_oracle import ray_set
from test_gpu_ray_mixer import _cuda, _make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first", [0, 5])
def test_gradients_with_states(first):
    """Rays looked at in two parts: values, states and the second part's gradients are those of one look along them."""
    R, T = 6, 26
    model, samples, features, _ = _make([T] * R)
    model, samples, features = model.cuda(), samples.cuda(), features.cuda()
    weight = torch.randn(R, T, 4, device="cuda")
    weight[:, :first] = 0.0  # the loss is of the second part
    whole_features = features.clone().requires_grad_()
    whole = model.look(samples, whole_features, _cuda(ray_set([T] * R)))
    (whole.view(R, T, 4) * weight).sum().backward()
    grads = {k: p.grad.clone() for k, p in model.named_parameters()}
    model.zero_grad()

    def part(t):
        t = t.view(R, T, -1)
        return t[:, :first].flatten(0, 1), t[:, first:].flatten(0, 1)

    state = model.states(R)
    with torch.no_grad():
        if first:
            model.look(part(samples)[0], part(features)[0], _cuda(ray_set([first] * R)), state)
    begun = state.clone()
    x = part(features)[1].clone().requires_grad_()
    y = model.look(part(samples)[1], x, _cuda(ray_set([T - first] * R)), state)
    assert y.requires_grad and not state.requires_grad
    (y.view(R, T - first, 4) * weight[:, first:]).sum().backward()
    # single precision in another order of sums: the bounds of the model's comparison with 64 bits, for both
    want = part(whole.detach())[1]
    assert float((y.detach() - want).abs().max()) < 2.0 ** -13 * max(1.0, float(want.abs().max()))
    want = part(whole_features.grad)[1]
    assert float((x.grad - want).abs().max()) < 2.0 ** -12 * float(want.abs().max())
    if not first:  # nothing before: all parameters have the same gradients
        for k, p in model.named_parameters():
            assert float((p.grad - grads[k]).abs().max()) < 2.0 ** -12 * float(grads[k].abs().max()) + 2.0 ** -19, k
    assert all(p.grad is not None for p in model.parameters())
    # the state is moved on as it is without gradients
    moved = state.clone()
    with torch.no_grad():
        model.look(part(samples)[1], x, _cuda(ray_set([T - first] * R)), begun)
    assert float((moved - begun).abs().max()) < 2.0 ** -13 * float(begun.abs().max())
