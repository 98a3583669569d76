"""Wrong arguments of layer norm and of routing: refused with a message, before any launch (nothing here reaches the
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
    _refused(lib.ffn_expert_slots, None, 100, 8, P, None, match="NULL plan")
    _refused(lib.ffn_expert_slots, P, 1 << 31, 8, P, None, match="exceed")
    _refused(lib.ffn_expert_slots, P, 100, 0, P, None, match="n_experts=0")


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
