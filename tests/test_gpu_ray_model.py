"""The ray model: the operators together, from the march to the composited colour and back."""
import pytest
import torch

from ray_oracle import ray_set

pytestmark = pytest.mark.gpu


def test_model_learns_the_ball():
    """The loss of the last steps is far below that of black images, the first steps' loss; two runs give the same bits."""
    import ray_model
    a = ray_model.train(steps=120, num_rays=512, seed=1)
    first, last = sum(a[:5]) / 5, sum(a[-10:]) / 10
    print(f"loss {first:.5f} -> {last:.5f}", flush=True)
    assert last < first / 10
    b = ray_model.train(steps=12, num_rays=512, seed=1)
    assert b == a[:12]


def test_model_matches_plain_operations():
    """Colour and gradients of the model in single precision against its formula in 64 bits (CPU, by automatic
    differentiation): rays of several lengths, one of them empty."""
    import ray_model
    import ray_ops
    torch.manual_seed(2)
    rays = ray_set([7, 0, 1, 20])
    n = rays[3]
    samples = torch.rand(n, 4)
    samples[:, 3] = torch.cat([torch.arange(int(c)) * 0.05 for c in rays[0]])
    features = torch.randn(n, 10)
    model = ray_model.RayModel(10, width=32, heads=2, dtype=torch.float32)
    torch.nn.init.normal_(model.b_1, std=0.3)
    weight = torch.randn(4, 3)

    def plain(m):
        d = {k: v.detach().double().requires_grad_() for k, v in m.named_parameters()}
        x = features.double() @ d["W_in"].T
        q, k, v = (x @ d["W_qkv"].T).view(n, 3, 2, 16).unbind(1)
        t = samples[:, 3].double()
        ids = rays[2].long()
        s = 30 * torch.tanh(torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0)) / 4 / 30)
        s = s - m.slopes.double()[:, None, None] * (t[:, None] - t[None, :]).abs()
        row = torch.arange(n)
        seen = (ids[:, None] == ids[None, :]) & (row[None, :] <= row[:, None])
        o = torch.softmax(s.masked_fill(~seen, -float("inf")), -1) @ v.transpose(0, 1)
        x = x + o.transpose(0, 1).reshape(n, -1) @ d["W_o"].T

        def scan(gate, x, order):
            out, states = [None] * n, []
            for r in range(4):
                h = torch.zeros(x.shape[1], dtype=torch.float64)
                o, c = int(rays[1][r]), int(rays[0][r])
                for i in (range(o, o + c) if order > 0 else range(o + c - 1, o - 1, -1)):
                    z = torch.sigmoid(gate[i])
                    h = (1 - z) * h + z * x[i]
                    out[i] = h
                states.append(h)
            return torch.stack(out), torch.stack(states)

        g, c = (x @ d["W_scan"].T).chunk(2, 1)
        x = x + scan(g, c, 1)[0]
        e = m.regions(samples).long()
        y = torch.relu(torch.matmul(d["W_1"][e], x[:, :, None])[..., 0] + d["b_1"][e])
        y = torch.matmul(d["W_2"][e], y[:, :, None])[..., 0] + d["b_2"][e]
        colour = scan(y[:, :1].expand(-1, 3), torch.sigmoid(y[:, 1:4]), -1)[1]
        (colour * weight.double()).sum().backward()
        return colour.detach(), {k: p.grad for k, p in d.items()}

    want, grads = plain(model)
    model = model.cuda()
    set_ = ray_ops.RaySet(*(x.cuda() for x in rays[:3]))
    colour = model(samples.cuda(), features.cuda(), set_)
    (colour * weight.cuda()).sum().backward()
    # some ten single precision operations in a row, each relative to its largest operands
    assert float((colour.detach().cpu().double() - want).abs().max()) < 2.0 ** -16
    for k, p in model.named_parameters():
        off = float((p.grad.cpu().double() - grads[k]).abs().max())
        assert off < 2.0 ** -15 * float(grads[k].abs().max()) + 2.0 ** -20, (k, off)
