"""Wrong arguments of layer norm, of routing and of the delta rule: refused with a message, before any launch (nothing here reaches the
GPU; pointers are never read)."""
import ctypes as C

import pytest

import ffn_lib as fl

P = 1 << 20  # a 16-byte aligned address that no call may touch


def _refused(fn, *args, match):
    assert fn(*args) == -1
    assert match in fl.load().ffn_last_error().decode(), fl.load().ffn_last_error()


def _norm(**kw):
    a = fl.FfnNorm(dtype=2, param_dtype=0, width=64, n=100, eps=1e-5, x=P, x_row=64, weight=P, bias=P, y=P, mean=P, rstd=P,
                   dy=P, dy_row=64, dx=P, dweight=P, dbias=P, workspace=P, workspace_bytes=1 << 30)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype=3"), (dict(param_dtype=1), "param_dtype=1"), (dict(width=0), "width=0"),
    (dict(width=fl.NORM_MAX_WIDTH + 1), "width=16385"), (dict(n=1 << 31), "exceed"), (dict(eps=-1.0), "eps=-1"),
    (dict(eps=float("nan")), "eps="), (dict(eps=float("inf")), "eps="), (dict(x=None), "NULL buffer"),
    (dict(mean=None), "NULL buffer"), (dict(rstd=None), "NULL buffer"), (dict(x=P + 1), "misaligned buffer"),
    (dict(weight=P + 2), "misaligned parameters"),
])
def test_norm_refuses(kw, match):
    lib = fl.load()
    _refused(lib.ffn_layer_norm_fwd, C.byref(_norm(**kw)), None, match=match)
    _refused(lib.ffn_layer_norm_bwd, C.byref(_norm(**kw)), None, match=match)


def test_norm_refuses_what_only_one_direction_needs():
    lib = fl.load()
    _refused(lib.ffn_layer_norm_fwd, C.byref(_norm(y=None)), None, match="NULL buffer")
    _refused(lib.ffn_layer_norm_bwd, C.byref(_norm(dy=None)), None, match="NULL buffer")
    _refused(lib.ffn_layer_norm_bwd, C.byref(_norm(workspace_bytes=64)), None, match="workspace of 64")
    _refused(lib.ffn_layer_norm_bwd, C.byref(_norm(workspace=None)), None, match="workspace of 0")
    _refused(lib.ffn_layer_norm_workspace, C.byref(_norm()), None, match="NULL bytes")
    _refused(lib.ffn_layer_norm_fwd, None, None, match="NULL arguments")


def _route(**kw):
    a = fl.FfnRoute(dtype=2, n_experts=8, k=2, width=64, n=100, plan=P, slots=P, weights=P, rows_in=P, rows_stride=64,
                    slots_in=P, slots_stride=64, rows_out=P, slots_out=P, dweights=P)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=-1), "dtype=-1"), (dict(k=0), "k=0"), (dict(k=1025), "k=1025"), (dict(width=0), "width=0"),
    (dict(width=65537), "width=65537"), (dict(n_experts=0), "n_experts=0"), (dict(n_experts=1025), "n_experts=1025"),
    (dict(n=1 << 30), "2147483648 places"), (dict(plan=None), "NULL plan"), (dict(slots=None), "NULL plan or slots"),
    (dict(rows_stride=-1), "strides"), (dict(slots_stride=-64), "strides"), (dict(rows_in=P + 1), "misaligned"),
    (dict(slots_out=P + 3), "misaligned"),
])
def test_route_refuses(kw, match):
    lib = fl.load()
    for fn in (lib.ffn_expert_dispatch, lib.ffn_expert_combine, lib.ffn_expert_combine_bwd):
        _refused(fn, C.byref(_route(**kw)), None, match=match)


def test_route_refuses_what_only_one_call_needs():
    lib = fl.load()
    _refused(lib.ffn_expert_dispatch, C.byref(_route(rows_in=None)), None, match="NULL buffer")
    _refused(lib.ffn_expert_dispatch, C.byref(_route(slots_out=None)), None, match="NULL buffer")
    _refused(lib.ffn_expert_combine, C.byref(_route(slots_in=None)), None, match="NULL buffer")
    _refused(lib.ffn_expert_combine, C.byref(_route(rows_out=None)), None, match="NULL buffer")
    _refused(lib.ffn_expert_combine_bwd, C.byref(_route(slots_in=None)), None, match="NULL buffer")
    _refused(lib.ffn_expert_combine_bwd, None, None, match="NULL arguments")
    _refused(lib.ffn_expert_route, None, 100, 8, P, 1 << 20, P, P, 1 << 20, None, match="NULL ids")
    _refused(lib.ffn_expert_route, P, 100, 8, P, 1 << 20, None, P, 1 << 20, None, match="NULL slots")
    _refused(lib.ffn_expert_route, P, 100, 8, P, 10, P, P, 1 << 20, None, match="plan of 10 words")
    _refused(lib.ffn_expert_route, P, 100000, 8, P, 1 << 20, P, P, 4, None, match="workspace of 4")
    _refused(lib.ffn_expert_route, P, 1 << 31, 8, P, 1 << 20, P, P, 1 << 20, None, match="exceed")
    _refused(lib.ffn_expert_route, P, 100, 0, P, 1 << 20, P, P, 1 << 20, None, match="n_experts=0")


def test_python_entry_points_refuse():
    import torch
    import ray_ops
    x = torch.zeros(4, 8)
    with pytest.raises(fl.FfnError, match="on the GPU"):
        ray_ops.layer_norm(x)
    with pytest.raises(fl.FfnError, match="on the GPU"):
        ray_ops.expert_route(torch.zeros(4, 2, dtype=torch.int32), 3)
    with pytest.raises(fl.FfnError, match="route must be a ExpertRoute"):
        ray_ops.expert_dispatch(x, None)


def _delta(**kw):
    s = dict(counts=P, offsets=P, ray_ids=P, num_rays=4, n=64)
    a = fl.FfnRayDelta(dtype=2, heads=2, v_heads=4, key_dim=32, val_dim=64, scale=0.2, rays=fl.FfnRaySet(**s), q=P, k=P, v=P,
                       q_row=64, q_head=32, k_row=64, k_head=32, v_row=256, v_head=64, decay=P, beta=P, decay_row=4,
                       decay_head=1, beta_row=4, beta_head=1, h0=P, o=P, last=P, marks=P, dout=P, do_row=256, do_head=64,
                       dlast=P, dq=P, dk=P, dv=P, ddecay=P, dbeta=P, dh0=P, workspace=P, workspace_bytes=1 << 30)
    for k, v in kw.items():
        setattr(a, k, fl.FfnRaySet(**{**s, **v}) if k == "rays" else v)
    return a


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype=3"), (dict(heads=3), "multiple of heads"), (dict(heads=0), "heads=0"),
    (dict(v_heads=1026), "v_heads=1026"), (dict(key_dim=12), "key_dim=12"), (dict(key_dim=136), "key_dim=136"),
    (dict(val_dim=0), "val_dim=0"), (dict(reverse=2), "reverse=2"), (dict(scale=float("nan")), "scale="),
    (dict(scale=float("inf")), "scale="), (dict(rays=dict(n=1 << 31)), "exceed"), (dict(rays=dict(counts=None)), "NULL counts"),
    (dict(rays=dict(ray_ids=None)), "NULL ray_ids"), (dict(rays=dict(num_rays=(1 << 32) - 1), v_heads=32), "2^36"),
    (dict(q=None), "NULL buffer"), (dict(beta=None), "NULL buffer"), (dict(q=P + 2), "aligned"), (dict(k_row=65), "aligned"),
    (dict(v_head=4), "aligned"), (dict(q_row=-64), "strides"), (dict(decay_head=-1), "strides"), (dict(k_row=1 << 23), "strides"), (dict(decay=P + 1), "misaligned"),
    (dict(h0=P + 4), "h0 must"), (dict(marks=P + 4), "16-byte aligned"),
])
def test_delta_refuses(kw, match):
    lib = fl.load()
    _refused(lib.ffn_ray_delta_fwd, C.byref(_delta(**kw)), None, match=match)
    _refused(lib.ffn_ray_delta_bwd, C.byref(_delta(**kw)), None, match=match)


def test_delta_refuses_what_only_one_direction_needs():
    lib = fl.load()
    _refused(lib.ffn_ray_delta_fwd, C.byref(_delta(o=None)), None, match="NULL output")
    _refused(lib.ffn_ray_delta_fwd, C.byref(_delta(last=P + 8)), None, match="16-byte aligned")
    for kw, match in ((dict(dout=None), "NULL gradient"), (dict(ddecay=None), "NULL gradient"), (dict(marks=None), "marks"),
                      (dict(do_row=4), "aligned"), (dict(dq=P + 8), "aligned"), (dict(do_row=-8), "strides"),
                      (dict(workspace_bytes=8), "workspace of 8"), (dict(workspace=None), "workspace of 0")):
        _refused(lib.ffn_ray_delta_bwd, C.byref(_delta(**kw)), None, match=match)
    _refused(lib.ffn_ray_delta_fwd, None, None, match="NULL arguments")
    _refused(lib.ffn_ray_delta_marks, C.byref(_delta()), None, match="NULL bytes")
    _refused(lib.ffn_ray_delta_workspace, C.byref(_delta()), 1, None, match="NULL bytes")
