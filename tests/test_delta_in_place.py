"""States that are written over those they start from: in place as a whole, and without a backward pass, or not at all."""
import ctypes as C

import pytest

import ffn_lib as fl
from test_more_refusals import P, _delta, _refused

SIZE = 4 * 4 * 32 * 64 * 4  # bytes of the states of _delta


def test_in_place_with_marks():
    _refused(fl.load().ffn_ray_delta_fwd, C.byref(_delta()), None, match="last is h0, and marks")


@pytest.mark.parametrize("by", [16, -16, 2 * SIZE // 4, 16 - SIZE, SIZE - 16])
@pytest.mark.parametrize("marks", [None, P])
def test_overlap(by, marks):
    _refused(fl.load().ffn_ray_delta_fwd, C.byref(_delta(last=P + by, marks=marks)), None, match="overlaps h0")


def test_python_entry_point():
    """Refused by the call that users make, before any launch: the rows here are on the GPU in name only."""
    import torch
    import ray_ops
    x = torch.zeros(3, 1, 8)

    class Rays(ray_ops.RaySet):
        def __init__(self):  # three rays of a row each, on no device (-1), as the tensors
            self.c = fl.FfnRaySet(counts=P, offsets=P, ray_ids=P, num_rays=3, n=3)
            self.num_rays, self.n, self.device = 3, 3, -1

    state = torch.zeros(4, 1, 8, 8)
    called = []

    def call(fn, dev, a):
        called.append(fn.__name__)
        fl.check(fn(a, None), fn.__name__)

    before, ray_ops._call = ray_ops._call, call
    empty, torch.empty = torch.empty, lambda *a, device=None, **k: empty(*a, **k)
    try:
        for kw, match in ((dict(h0=state[:3], last=state[:3], marks=True), "last is h0"),
                          (dict(h0=state[:3], last=state[1:]), "overlaps h0")):
            with pytest.raises(fl.FfnError, match=match):
                ray_ops.ray_delta(x, x, x, x[:, :, 0], x[:, :, 0], Rays(), **kw)
    finally:
        ray_ops._call, torch.empty = before, empty
    assert called == ["ffn_ray_delta_fwd"] * 2
