"""Buffers of 4-byte values that start between two of them: refused by norm and routing, before any launch."""
import ctypes as C

import pytest

import ffn_lib as fl
from test_more_refusals import P, _norm, _refused, _route


@pytest.mark.parametrize("by", [1, 2, 3])
@pytest.mark.parametrize("name", ["mean", "rstd", "dweight", "dbias"])
def test_norm(name, by):
    lib = fl.load()
    for fn in (lib.ffn_layer_norm_fwd, lib.ffn_layer_norm_bwd):
        _refused(fn, C.byref(_norm(**{name: P + by})), None, match="misaligned mean, rstd, dweight or dbias")


@pytest.mark.parametrize("by", [1, 2, 3])
@pytest.mark.parametrize("name", ["plan", "slots", "weights", "dweights"])
def test_route(name, by):
    lib = fl.load()
    for fn in (lib.ffn_expert_dispatch, lib.ffn_expert_combine, lib.ffn_expert_combine_bwd):
        _refused(fn, C.byref(_route(**{name: P + by})), None, match="misaligned plan, slots, weights or dweights")


def test_making_a_route():
    fn = fl.load().ffn_expert_route
    _refused(fn, P + 2, 100, 8, P, 1 << 20, P, P, 1 << 20, None, match="misaligned ids or slots")
    _refused(fn, P, 100, 8, P, 1 << 20, P + 1, P, 1 << 20, None, match="misaligned ids or slots")
