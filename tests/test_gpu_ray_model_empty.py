"""The ray model on a batch whose rays all miss."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_all_rays_miss(dtype):
    """Black rays, and gradients of 0."""
    import ray_model
    import ray_ops
    zeros = torch.zeros(5, dtype=torch.int32, device="cuda")
    rays = ray_ops.RaySet(zeros, zeros, zeros[:0])
    model = ray_model.RayModel(10, width=32, heads=2, dtype=dtype).cuda()
    features = torch.empty(0, 10, device="cuda", requires_grad=True)
    colour = model(torch.empty(0, 4, device="cuda"), features, rays)
    assert colour.shape == (5, 3) and not colour.any()
    ((colour - 1.0) ** 2).mean().backward()
    assert features.grad.shape == (0, 10)
    for name, p in model.named_parameters():
        assert p.grad is not None and not p.grad.any(), name


def test_march_that_finds_nothing(tmp_path):
    """From an empty bitfield to the loss's gradient in the hash table."""
    import numpy as np
    import ffnerf_tools as ft
    import ray_model
    import synthetic_scene as scene
    spec = ft.ModelSpec(n_levels=4, f_per_level=2, log2_T=[12] * 4, res=ft.level_resolutions(4, 16.0, growth=1.5))
    nerf = ft.Nerf(str(tmp_path), "rays", spec=spec, occ=ft.OccParams(G_occ=16, box_min=np.zeros(3), box_max=np.ones(3)))
    rays, _ = scene.uniform_batch(scene.cameras_for("cfg0", seed=0), 40, np.random.default_rng(0))
    rays = torch.from_numpy(ft.rays_as_array(rays)).cuda()
    bits = torch.zeros(32 ** 3 // 32, dtype=torch.int32, device="cuda")
    samples, ray_set = ray_model.march_samples(nerf, rays, bits, 32, 0.03, 64)
    assert samples.shape[0] == 0
    table = torch.nn.Parameter(nerf.t["table"])
    xyz = samples[:, :3].contiguous()
    features = torch.cat((ray_model.HashEncode.apply(table, xyz, nerf), xyz), 1)
    colour = ray_model.RayModel(spec.lf + 3).cuda()(samples, features, ray_set)
    assert colour.shape == (40, 3) and not colour.any()
    (colour ** 2).sum().backward()
    assert not table.grad.any()
