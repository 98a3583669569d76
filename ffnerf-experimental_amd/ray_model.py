"""Models that look along their rays, on the operators of ray_ops: examples that train, and modules to start from.

`march_samples` takes a batch's samples from the occupancy bitfield, `HashEncode` encodes them.  `RayModel` then lets the samples of
a ray attend to those in front of them (ray_attention: causal in the ray's order, scores that fall with the distance in
depth), carries features along the ray (ray_scan), sends every sample through the layers of its region of the box
(expert_plan, expert_linear) and composites opacity and colour back to front (ray_scan again).  `RayMixer` is a block of the
other kind: normalised features (layer_norm), a matrix of what the ray has shown so far (ray_delta), and the layers of a
sample's own region and of the nearest other one, blended (expert_route, expert_dispatch, expert_combine); it can be asked
sample by sample, with the rays' states in hand.

    python ffnerf-experimental_amd/ray_model.py --steps 200 [--model mixer]     # the synthetic ball scene
"""
from __future__ import annotations

import argparse
import ctypes as C
import sys
import tempfile

import numpy as np
import torch

import ffn_lib as fl
from ray_ops import (ExpertCombine, ExpertDispatch, ExpertLinear, LayerNorm, RayAttention, RayDelta, RayScan, RaySet,
                     expert_plan, expert_route, once, ray_delta)


class HashEncode(torch.autograd.Function):
    """Features [n, LF] of positions xyz [n, 3] from the hash table of `nerf`; differentiable in the table, which is
    nerf.t["table"] itself (an optimizer that updates it in place trains it)."""

    @staticmethod
    def forward(ctx, table, xyz, nerf):
        a0 = torch.empty((xyz.shape[0], nerf.spec.lf), dtype=torch.float32, device=xyz.device)
        fl.check(nerf.handle.lib.ffn_hash_encode_fwd(nerf.handle.h, fl.ptr(xyz), xyz.shape[0], fl.ptr(a0), None,
                                                     fl.stream_ptr()), "ffn_hash_encode_fwd")
        ctx.save_for_backward(xyz)
        ctx.nerf = nerf
        return a0

    @staticmethod
    def backward(ctx, g):
        xyz, = ctx.saved_tensors
        nerf = ctx.nerf

        def grad():
            to, rows = torch.zeros_like(nerf.t["table"]), g.contiguous()
            fl.check(nerf.handle.lib.ffn_hash_encode_bwd(nerf.handle.h, fl.ptr(xyz), fl.ptr(rows), xyz.shape[0],
                                                         fl.ptr(to), fl.stream_ptr()), "ffn_hash_encode_bwd")
            return to

        return once(grad, g), None, None


def march_samples(nerf, rays, bits, res: int, dt: float, max_steps: int):
    """(samples [n, 4] {x, y, z, t}, RaySet) of rays [num_rays, 8] marched through a bitfield.  Waits once, for the number
    of samples."""
    lib, n = nerf.handle.lib, rays.shape[0]
    cap = n * max_steps
    counts, offsets, total = (torch.empty(k, dtype=torch.int32, device=rays.device) for k in (n, n, 4))
    samples = torch.empty((cap, 4), dtype=torch.float32, device=rays.device)
    ids = torch.empty(cap, dtype=torch.int32, device=rays.device)
    mp = fl.march_params(res, dt, max_steps)
    fl.check(lib.ffn_march(nerf.handle.h, fl.ptr(rays), n, fl.ptr(bits), C.byref(mp), fl.ptr(counts), fl.ptr(offsets),
                           fl.ptr(samples), fl.ptr(ids), cap, fl.ptr(total), fl.stream_ptr()), "ffn_march")
    m = int(total[0].item())
    return samples[:m], RaySet(counts, offsets, ids[:m])


class RayModel(torch.nn.Module):
    """features: width of the samples' features; cells: regions of the box an axis, each with expert layers of its own;
    dtype: of the operators (the parameters stay float32)."""

    def __init__(self, features: int, width: int = 64, heads: int = 4, cells: int = 2, box=((0.0,) * 3, (1.0,) * 3),
                 dtype=torch.bfloat16):
        super().__init__()
        if width % (8 * heads):
            raise ValueError(f"width={width} must be a multiple of 8 heads={heads}")
        self.width, self.heads, self.cells, self.dtype, experts = width, heads, cells, dtype, cells ** 3

        def weight(*shape):
            return torch.nn.Parameter(torch.randn(shape) * shape[-1] ** -0.5)

        self.W_in, self.W_qkv, self.W_o = weight(width, features), weight(3 * width, width), weight(width, width)
        self.W_scan = weight(2 * width, width)
        self.W_1, self.b_1 = weight(experts, width, width), torch.nn.Parameter(torch.zeros(experts, width))
        self.W_2, self.b_2 = weight(experts, 8, width), torch.nn.Parameter(torch.zeros(experts, 8))
        self.register_buffer("slopes", torch.tensor([8.0 * 2.0 ** -h for h in range(heads)]))
        self.register_buffer("lo", torch.tensor(box[0]))
        self.register_buffer("hi", torch.tensor(box[1]))

    def regions(self, samples) -> torch.Tensor:
        """The expert of each sample: the cell of the box that holds it."""
        c = ((samples[:, :3] - self.lo) / (self.hi - self.lo) * self.cells).long().clamp(0, self.cells - 1)
        return ((c[:, 2] * self.cells + c[:, 1]) * self.cells + c[:, 0]).to(torch.int32)

    def forward(self, samples, features, rays: RaySet) -> torch.Tensor:
        """Colour [num_rays, 3] of each ray on a black background."""
        t, n, ty = samples[:, 3], samples.shape[0], self.dtype
        x = (features @ self.W_in.t()).to(ty)
        qkv = (x @ self.W_qkv.to(ty).t()).view(n, 3, self.heads, self.width // self.heads)
        o = RayAttention.apply(qkv[:, 0], qkv[:, 1], qkv[:, 2], rays, None,
                               dict(t_q=t, t_k=t, slopes=self.slopes, cap=30.0, causal=True))
        x = x + o.reshape(n, self.width) @ self.W_o.to(ty).t()
        gate, carry = (x @ self.W_scan.to(ty).t()).chunk(2, 1)
        x = x + RayScan.apply(gate, carry, rays)[0]
        plan = expert_plan(self.regions(samples), self.cells ** 3)
        y = ExpertLinear.apply(x, self.W_1.to(ty), self.b_1.to(ty), plan, True, False, True)
        y = ExpertLinear.apply(y, self.W_2.to(ty), self.b_2.to(ty), plan, False, True, False).float()
        opacity = y[:, :1].expand(-1, 3).contiguous()
        return RayScan.apply(opacity, torch.sigmoid(y[:, 1:4]), rays, None, True)[1]


class RayMixer(torch.nn.Module):
    """features: width of the samples' features; cells: regions of the box an axis, each with expert layers of its own;
    dtype: of the operators (the parameters stay float32)."""

    def __init__(self, features: int, width: int = 64, heads: int = 4, cells: int = 2, box=((0.0,) * 3, (1.0,) * 3),
                 dtype=torch.bfloat16):
        super().__init__()
        if width % (8 * heads):
            raise ValueError(f"width={width} must be a multiple of 8 heads={heads}")
        self.width, self.heads, self.cells, self.dtype, experts = width, heads, cells, dtype, cells ** 3

        def weight(*shape):
            return torch.nn.Parameter(torch.randn(shape) * shape[-1] ** -0.5)

        def norm():
            return torch.nn.Parameter(torch.ones(width)), torch.nn.Parameter(torch.zeros(width))

        self.W_in, self.W_qkv, self.W_o = weight(width, features), weight(3 * width, width), weight(width, width)
        self.W_gates, self.b_gates = weight(2 * heads, width), torch.nn.Parameter(torch.tensor([-3.0] * heads + [0.0] * heads))
        self.W_1, self.b_1 = weight(experts, width, width), torch.nn.Parameter(torch.zeros(experts, width))
        self.W_2, self.b_2 = weight(experts, width, width), torch.nn.Parameter(torch.zeros(experts, width))
        self.W_out, self.b_out = weight(4, width), torch.nn.Parameter(torch.zeros(4))
        (self.n_1, self.m_1), (self.n_2, self.m_2), (self.n_3, self.m_3) = norm(), norm(), norm()
        self.register_buffer("lo", torch.tensor(box[0]))
        self.register_buffer("hi", torch.tensor(box[1]))

    def blend(self, samples):
        """(ids [n, 2], weights [n, 2]): the region of each sample and the one across the nearest face, which has half the
        weight at that face and none at the centre; -1 where the face is the box's own."""
        u = ((samples[:, :3] - self.lo) / (self.hi - self.lo) * self.cells).clamp(0, self.cells)
        c = u.floor().clamp(max=self.cells - 1)
        off = u - c - 0.5
        far, axis = off.abs().max(1)
        to = torch.gather(c, 1, axis[:, None])[:, 0] + torch.sign(torch.gather(off, 1, axis[:, None])[:, 0])
        other = c.scatter(1, axis[:, None], to[:, None])
        inside = (to >= 0) & (to < self.cells) & (far > 0)
        ids = torch.stack([(x[:, 2] * self.cells + x[:, 1]) * self.cells + x[:, 0] for x in (c, other)], 1).to(torch.int32)
        ids[:, 1] = torch.where(inside, ids[:, 1], -1)
        w = torch.where(inside, far.clamp(max=0.5), 0.0)
        return ids, torch.stack((1 - w, w), 1)

    def states(self, num_rays: int) -> torch.Tensor:
        """States of rays of which nothing has been seen."""
        d = self.width // self.heads
        return torch.zeros(num_rays, self.heads, d, d, device=self.lo.device)

    def look(self, samples, features, rays: RaySet, state=None):
        """Opacity and colour, before their sigmoids, of each sample [n, 4] from it and those in front of it.  state: what
        the rays have shown before these samples; it is moved on in place.  Gradients are those of these samples: none
        passes through the state to the ones before them."""
        n, ty, d = samples.shape[0], self.dtype, self.width // self.heads
        x = (features @ self.W_in.t()).to(ty)
        h = LayerNorm.apply(x, self.n_1, self.m_1)
        q, k, v = (h @ self.W_qkv.to(ty).t()).view(n, 3, self.heads, d).unbind(1)
        q, k = (torch.nn.functional.normalize(t.float(), dim=-1).to(ty) for t in (q, k))
        decay, beta = (h.float() @ self.W_gates.t() + self.b_gates).chunk(2, 1)
        decay, beta = -torch.nn.functional.softplus(decay).to(ty), torch.sigmoid(beta).to(ty)
        if state is None:
            o = RayDelta.apply(q, k, v, decay, beta, rays, None, dict(last=False))[0]
        elif torch.is_grad_enabled():
            o, last = RayDelta.apply(q, k, v, decay, beta, rays, state.detach().clone())  # kept for the backward
            with torch.no_grad():
                state.copy_(last)
        else:
            o = ray_delta(q, k, v, decay, beta, rays, h0=state, last=state)[0]
        x = x + o.reshape(n, self.width) @ self.W_o.to(ty).t()
        ids, weights = self.blend(samples)
        route = expert_route(ids, self.cells ** 3)
        y = ExpertDispatch.apply(LayerNorm.apply(x, self.n_2, self.m_2), route)
        y = ExpertLinear.apply(y, self.W_1.to(ty), self.b_1.to(ty), route.plan, True, True, True)
        y = ExpertLinear.apply(y, self.W_2.to(ty), self.b_2.to(ty), route.plan, False, True, True)
        x = x + ExpertCombine.apply(y, route, weights)
        return LayerNorm.apply(x, self.n_3, self.m_3).float() @ self.W_out.t() + self.b_out

    def forward(self, samples, features, rays: RaySet) -> torch.Tensor:
        """Colour [num_rays, 3] of each ray on a black background."""
        y = self.look(samples, features, rays)
        opacity = y[:, :1].expand(-1, 3).contiguous()
        return RayScan.apply(opacity, torch.sigmoid(y[:, 1:4]), rays, None, True)[1]


MODELS = {"attend": RayModel, "mixer": RayMixer}


def train(steps: int = 200, num_rays: int = 1024, lr: float = 3e-3, seed: int = 0, report=None, model: str = "attend") -> list:
    """Trains a model of MODELS on rays of the synthetic ball scene; the loss of each step."""
    import ffnerf_tools as ft
    import synthetic_scene as scene
    torch.manual_seed(seed)
    rng = np.random.default_rng(seed)
    spec = ft.ModelSpec(n_levels=8, f_per_level=2, log2_T=[14] * 8, res=ft.level_resolutions(8, 16.0, growth=1.5))
    occ = ft.OccParams(G_occ=16, box_min=np.zeros(3), box_max=np.ones(3))
    R, dt, max_steps = 32, float(np.float32(np.sqrt(3.0) / 64)), 64
    c = (np.arange(R) + 0.5) / R
    z, y, x = np.meshgrid(c, c, c, indexing="ij")
    ball = (x - 0.5) ** 2 + (y - 0.5) ** 2 + (z - 0.5) ** 2 < 0.3 ** 2
    bits = torch.from_numpy(np.packbits(ball.reshape(-1), bitorder="little").view(np.int32).copy()).cuda()
    cams = scene.cameras_for("cfg0", seed=seed)
    losses = []
    with tempfile.TemporaryDirectory() as d:
        nerf = ft.Nerf(d, "rays", spec=spec, occ=occ)
        net = MODELS[model](spec.lf + 3).cuda()
        table = torch.nn.Parameter(nerf.t["table"])  # the same memory: what the handle reads
        adam = torch.optim.Adam([dict(params=net.parameters(), lr=lr), dict(params=[table], lr=10 * lr, eps=1e-15)])
        for step in range(steps):
            rays, targets = scene.uniform_batch(cams, num_rays, rng)
            rays = torch.from_numpy(ft.rays_as_array(rays)).cuda()
            want = torch.from_numpy(np.asarray(targets, np.float32)[:, :3].copy()).cuda()
            samples, ray_set = march_samples(nerf, rays, bits, R, dt, max_steps)
            xyz = samples[:, :3].contiguous()
            colour = net(samples, torch.cat((HashEncode.apply(table, xyz, nerf), xyz), 1), ray_set)
            loss = ((colour - want) ** 2).mean()
            adam.zero_grad()
            loss.backward()
            adam.step()
            losses.append(loss.detach())
            if report and (step % 20 == 0 or step == steps - 1):
                report(f"step {step}  loss {float(losses[-1]):.6f}  samples {samples.shape[0]}")
    return [float(v) for v in losses]


def main(argv=None) -> int:
    p = argparse.ArgumentParser(description="Train a model that looks along its rays on the synthetic ball scene.")
    p.add_argument("--steps", type=int, default=200)
    p.add_argument("--rays", type=int, default=1024)
    p.add_argument("--model", choices=sorted(MODELS), default="attend")
    args = p.parse_args(argv)
    train(args.steps, args.rays, model=args.model, report=lambda s: print(s, flush=True))
    return 0


if __name__ == "__main__":
    sys.exit(main())
