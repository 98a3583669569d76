"""Strides of the delta rule's arguments: rows less than 2^24 bytes apart, heads any way apart, neither below 0."""
import ctypes as C

import pytest

import ffn_lib as fl
from test_more_refusals import P, _delta, _refused

ROWS, HEADS = ["q_row", "k_row", "v_row", "decay_row", "beta_row"], ["q_head", "k_head", "v_head", "decay_head", "beta_head"]


@pytest.mark.parametrize("name", ROWS + ["do_row"])
def test_rows(name):
    lib = fl.load()
    for stride in (1 << 23, -64):
        a = C.byref(_delta(**{name: stride}))
        _refused(lib.ffn_ray_delta_bwd, a, None, match="row strides")
        if name != "do_row":
            _refused(lib.ffn_ray_delta_fwd, a, None, match="row strides")


@pytest.mark.parametrize("name", HEADS + ["do_head"])
def test_heads(name):
    lib = fl.load()
    a = C.byref(_delta(**{name: -64}))
    _refused(lib.ffn_ray_delta_bwd, a, None, match="head strides")
    # a far head is no reason to refuse: what is refused here is the buffer that is looked at after it
    far = C.byref(_delta(**{name: 1 << 30}, h0=P + 4))
    _refused(lib.ffn_ray_delta_fwd, far, None, match="h0 must")
    _refused(lib.ffn_ray_delta_bwd, far, None, match="h0 must")
