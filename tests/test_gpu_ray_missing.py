"""Arguments that are missing or of the wrong kind: an FfnError that names them, from every entry point on tensors."""
import pytest
import torch

from ray_oracle import ray_set

pytestmark = pytest.mark.gpu


def _calls():
    """Each entry point with arguments that it takes, by name."""
    import ray_ops
    rays = ray_ops.RaySet(*(x.cuda() for x in ray_set([4, 3])[:3]))
    x, z = torch.randn(7, 2, 16, device="cuda"), torch.randn(7, 8, device="cuda")
    o, lse = ray_ops.ray_attention(x, x, x, rays)
    _, _, marks = ray_ops.ray_scan(z, z, rays, marks=True)
    plan = ray_ops.expert_plan(torch.zeros(7, dtype=torch.int32, device="cuda"), 2)
    W = torch.randn(2, 16, 8, device="cuda")
    options = dict(t_q=x[:, 0, 0], t_k=x[:, 0, 0], slopes=x[0, :, 0].contiguous(), scale=0.5, cap=1.0, causal=True,
                   prefix=torch.zeros(2, dtype=torch.int32, device="cuda"))
    return {
        "ray_attention": dict(q=x, k=x, v=x, q_rays=rays, k_rays=rays, **options),
        "ray_attention_backward": dict(do=x, q=x, k=x, v=x, o=o, lse=lse, q_rays=rays, k_rays=rays, **options),
        "ray_scan": dict(gate=z, x=z, rays=rays, h0=z[:2]),
        "ray_scan_backward": dict(dh=z, gate=z, x=z, marks=marks, rays=rays, dlast=z[:2], h0=z[:2]),
        "expert_plan": dict(ids=torch.zeros(7, dtype=torch.int32, device="cuda"), n_experts=2),
        "expert_linear": dict(x=z, W=W, b=W[:, :, 0].contiguous(), plan=plan),
        "expert_linear_backward": dict(dy=torch.randn(7, 16, device="cuda"), x=z, W=W, plan=plan, y=torch.randn(7, 16, device="cuda")),
    }


OPTIONAL = {"k_rays", "slopes", "scale", "prefix", "h0", "dlast", "b", "y", "causal"}
NAMES = ["ray_attention", "ray_attention_backward", "ray_scan", "ray_scan_backward", "expert_plan", "expert_linear",
         "expert_linear_backward"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("wrong", [None, [1.0, 2.0], "text"], ids=["none", "list", "text"])
def test_wrong_kinds(name, wrong):
    import ffn_lib as fl
    import ray_ops
    args = _calls()[name]
    getattr(ray_ops, name)(**args)
    for which in args:
        if which == "causal" or wrong is None and which in OPTIONAL:
            continue
        with pytest.raises(fl.FfnError) as e:
            getattr(ray_ops, name)(**{**args, which: wrong})
        assert which in str(e.value), (which, str(e.value))


def test_numbers_out_of_range():
    import ffn_lib as fl
    import ray_ops
    ids = torch.zeros(7, dtype=torch.int32, device="cuda")
    for n in (0, -1, 1025, 2 ** 32 + 2, 2.0):
        with pytest.raises(fl.FfnError, match="n_experts"):
            ray_ops.expert_plan(ids, n)
    args = _calls()["ray_attention"]
    for name, value in (("scale", float("inf")), ("scale", 1e300), ("cap", -1.0), ("cap", float("nan"))):
        with pytest.raises(fl.FfnError, match=name):
            ray_ops.ray_attention(**{**args, name: value})
