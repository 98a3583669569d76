"""Sizes past what a launch can count are refused (nothing here reaches the GPU; pointers are never read)."""
import ctypes as C

import ffn_lib as fl

P = 1 << 20  # a 16-byte aligned address that no call may touch


def test_recurrence_of_too_many_states():
    lib = fl.load()
    a = fl.FfnRayScan(dtype=0, channels=65536, rays=fl.FfnRaySet(counts=P, offsets=P, ray_ids=P, num_rays=(1 << 30) + 1, n=64),
                      gate=P, x=P, gate_row=65536, x_row=65536, h=P, marks=P, dh=P, dh_row=65536, dgate=P, dx=P, workspace=P,
                      workspace_bytes=1 << 60)
    for fn in (lib.ffn_ray_scan_fwd, lib.ffn_ray_scan_bwd):
        assert fn(C.byref(a), None) == -1
        assert "2^46" in lib.ffn_last_error().decode()
