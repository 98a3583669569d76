"""Wrong arguments of the operators along rays and of the expert layers: refused with a message, before any launch
(nothing here reaches the GPU; pointers are never read)."""
import ctypes as C

import pytest

import ffn_lib as fl

P = 1 << 20  # a 16-byte aligned address that no call may touch


def _attn(**kw):
    s = dict(counts=P, offsets=P, ray_ids=P, num_rays=4, n=64)
    a = fl.FfnRayAttn(dtype=2, heads=4, kv_heads=2, dim=32, scale=0.1, cap=0.0, causal=1, q_rays=fl.FfnRaySet(**s),
                      k_rays=fl.FfnRaySet(**s), q=P, k=P, v=P, q_row=128, q_head=32, k_row=64, k_head=32, v_row=64,
                      v_head=32, o=P, lse=P, dout=P, do_row=128, do_head=32, dq=P, dk=P, dv=P, workspace=P,
                      workspace_bytes=1 << 30)
    for k, v in kw.items():
        if k in ("q_rays", "k_rays"):
            setattr(a, k, fl.FfnRaySet(**{**s, **v}))
        else:
            setattr(a, k, v)
    return a


def _refused(fn, *args, match):
    assert fn(*args) < 0
    assert match in fl.load().ffn_last_error().decode(), fl.load().ffn_last_error()


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype=3"), (dict(heads=3), "multiple of kv_heads"), (dict(kv_heads=0), "kv_heads=0"),
    (dict(dim=12), "dim=12"), (dict(dim=136), "dim=136"), (dict(dim=0), "dim=0"), (dict(cap=-1.0), "cap=-1"),
    (dict(cap=float("nan")), "cap="), (dict(scale=float("inf")), "scale="), (dict(q=None), "NULL buffer"),
    (dict(v=None), "NULL buffer"), (dict(lse=None), "NULL buffer"), (dict(q=P + 2), "aligned"),
    (dict(k_row=65), "aligned"), (dict(v_head=4), "aligned"), (dict(slopes=P), "t_q"),
    (dict(q_rays=dict(num_rays=5)), "queries of 5 rays"), (dict(k_rays=dict(n=1 << 31)), "exceed"),
    (dict(q_rays=dict(counts=None)), "NULL counts"), (dict(q_rays=dict(ray_ids=None)), "NULL ray_ids"),
])
def test_attention_refuses(kw, match):
    lib = fl.load()
    _refused(lib.ffn_ray_attention_fwd, C.byref(_attn(**kw)), None, match=match)
    _refused(lib.ffn_ray_attention_bwd, C.byref(_attn(**kw)), None, match=match)


def test_attention_refuses_what_only_one_direction_needs():
    lib = fl.load()
    for kw, match in ((dict(dout=None), "NULL gradient"), (dict(dk=None), "NULL gradient"),
                      (dict(dq=P + 4), "aligned"), (dict(workspace_bytes=8), "workspace of 8"),
                      (dict(workspace=None), "workspace of 0"), (dict(k_rays=dict(ray_ids=None)), "NULL ray_ids")):
        _refused(lib.ffn_ray_attention_bwd, C.byref(_attn(**kw)), None, match=match)
    few = dict(q_rays=dict(n=2), k_rays=dict(n=4096), workspace_bytes=8)
    _refused(lib.ffn_ray_attention_fwd, C.byref(_attn(**few)), None, match="workspace of 8")
    _refused(lib.ffn_ray_attention_fwd, None, None, match="NULL arguments")
    _refused(lib.ffn_ray_attention_workspace, C.byref(_attn()), 0, None, match="NULL bytes")


def _scan(**kw):
    a = fl.FfnRayScan(dtype=0, channels=8, rays=fl.FfnRaySet(counts=P, offsets=P, ray_ids=P, num_rays=4, n=64), gate=P,
                      x=P, gate_row=8, x_row=8, h=P, marks=P, dh=P, dh_row=8, dgate=P, dx=P, workspace=P,
                      workspace_bytes=1 << 30)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=-1), "dtype=-1"), (dict(channels=0), "channels=0"), (dict(channels=65537), "channels=65537"),
    (dict(reverse=2), "reverse=2"), (dict(x_row=(1 << 25) + 1), "bytes apart"), (dict(x=None), "NULL buffer"), (dict(gate=P + 1), "misaligned"),
    (dict(rays=fl.FfnRaySet(num_rays=4, n=64, ray_ids=P)), "NULL counts"),
    (dict(rays=fl.FfnRaySet(counts=P, offsets=P, num_rays=4, n=64)), "NULL ray_ids"),
])
def test_scan_refuses(kw, match):
    lib = fl.load()
    _refused(lib.ffn_ray_scan_fwd, C.byref(_scan(**kw)), None, match=match)
    _refused(lib.ffn_ray_scan_bwd, C.byref(_scan(**kw)), None, match=match)


def test_scan_refuses_what_only_one_direction_needs():
    lib = fl.load()
    _refused(lib.ffn_ray_scan_fwd, C.byref(_scan(h=None)), None, match="NULL output")
    _refused(lib.ffn_ray_scan_bwd, C.byref(_scan(dx=None)), None, match="NULL gradient")
    _refused(lib.ffn_ray_scan_bwd, C.byref(_scan(marks=None)), None, match="marks")
    _refused(lib.ffn_ray_scan_bwd, C.byref(_scan(dh=P + 2)), None, match="misaligned")


def _experts(**kw):
    a = fl.FfnExperts(dtype=2, n_experts=4, d_in=64, d_out=32, relu=1, n=100, plan=P, x=P, x_row=64, W=P, b=P, y=P,
                      dy=P, dy_row=32, dx=P, dW=P, db=P, workspace=P, workspace_bytes=1 << 30)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=5), "dtype=5"), (dict(n_experts=0), "n_experts=0"), (dict(n_experts=1025), "n_experts=1025"),
    (dict(d_in=12), "in=12"), (dict(d_out=4104), "out=4104"), (dict(flags=4), "flags"), (dict(plan=None), "NULL plan"),
    (dict(x=None), "NULL buffer"), (dict(W=None), "NULL buffer"), (dict(y=None), "NULL buffer"),
    (dict(x_row=65), "aligned"), (dict(x_row=-64), "row strides"), (dict(dy_row=1 << 31), "row strides"),
    (dict(W=P + 8), "aligned"), (dict(n=(1 << 31)), "exceed"),
])
def test_experts_refuse(kw, match):
    lib = fl.load()
    _refused(lib.ffn_expert_linear_fwd, C.byref(_experts(**kw)), None, match=match)
    _refused(lib.ffn_expert_linear_bwd, C.byref(_experts(**kw)), None, match=match)


def test_experts_refuse_what_only_one_call_needs():
    lib = fl.load()
    _refused(lib.ffn_expert_linear_bwd, C.byref(_experts(dy=None)), None, match="NULL buffer")
    _refused(lib.ffn_expert_linear_bwd, C.byref(_experts(workspace_bytes=16)), None, match="workspace of 16")
    _refused(lib.ffn_expert_plan, P, 100, 4, P, 10, P, 1 << 20, None, match="plan of 10 words")
    _refused(lib.ffn_expert_plan, P, 100000, 4, P, 1 << 20, P, 4, None, match="workspace of 4")
    _refused(lib.ffn_expert_plan, None, 100, 4, P, 1 << 20, P, 1 << 20, None, match="NULL ids")
    _refused(lib.ffn_expert_plan_size, 100, 0, C.byref(C.c_uint64()), C.byref(C.c_uint64()), match="n_experts=0")


def test_python_entry_points_refuse():
    import torch
    import ray_ops
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(fl.FfnError, match="on the GPU"):
        ray_ops.RaySet(i, i, i)
    with pytest.raises(fl.FfnError, match="on the GPU"):
        ray_ops.expert_plan(i, 2)
