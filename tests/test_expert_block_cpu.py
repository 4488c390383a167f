"""Argument checks of the expert-block entry points (include/facedet.h), which come before any GPU call: bad shapes and
missing pointers are FD_ERR_ARG, documented limits FD_ERR_LIMIT, and an empty problem does nothing.  No GPU work."""
import ctypes as C

import pytest

from facedetection_amd import _lib

P = 4096          # a non-NULL pointer; every call below returns before it is used
ARG, LIMIT = -1, -3


def _err():
    return _lib.lib().fd_last_error().decode()


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), ARG), (dict(x_rows=-1), ARG), (dict(inner=0), ARG), (dict(experts=0), ARG), (dict(outputs=0), ARG), (dict(slots=-1), ARG),
    (dict(act=4), ARG), (dict(act=-1), ARG), (dict(rows=None, slots=9), ARG), (dict(weight=None), ARG), (dict(offsets=None), ARG),
    (dict(y=None), ARG), (dict(x=None), ARG), (dict(experts=1025), LIMIT), (dict(inner=(1 << 24) + 1), LIMIT),
    (dict(slots=(1 << 31) - 1024), LIMIT), (dict(slots=0), 0),
])
def test_expert_linear_refuses(change, code):
    a = dict(x=P, dtype=0, x_rows=8, inner=16, weight=P, experts=4, outputs=8, offsets=P, rows=P, slots=16, bias=None, act=0, gated=0, y=P)
    a.update(change)
    rc = _lib.lib().fd_expert_linear(a["x"], a["dtype"], a["x_rows"], a["inner"], a["weight"], a["experts"], a["outputs"], a["offsets"],
                                     a["rows"], a["slots"], a["bias"], a["act"], a["gated"], a["y"], None)
    assert rc == code and (rc == 0 or "fd_expert_linear" in _err())


@pytest.mark.parametrize("change,code", [
    (dict(dtype=-1), ARG), (dict(rows=-1), ARG), (dict(experts=0), ARG), (dict(k=0), ARG), (dict(k=9), ARG), (dict(logits=None), ARG),
    (dict(offsets=None), ARG), (dict(experts=513), LIMIT), (dict(experts=64, k=17), LIMIT), (dict(rows=1 << 31, k=1), LIMIT),
    (dict(rows=513, nbytes=0), ARG), (dict(rows=513, nbytes=63), ARG), (dict(rows=513, work=None, nbytes=64), ARG),
])
def test_expert_route_refuses(change, code):
    a = dict(logits=P, dtype=0, rows=10, experts=8, k=2, offsets=P, work=P, nbytes=1 << 40)
    a.update(change)
    rc = _lib.lib().fd_expert_route(a["logits"], a["dtype"], a["rows"], a["experts"], a["k"], None, 1, P, P, P, a["offsets"], P, a["work"],
                                    a["nbytes"], None)
    assert rc == code and "fd_expert_route" in _err()


def test_expert_route_workspace_is_for_more_than_one_workgroup():
    L = _lib.lib()
    assert L.fd_expert_route_workspace(0, 8) == 0 and L.fd_expert_route_workspace(512, 8) == 0
    assert L.fd_expert_route_workspace(513, 8) == 2 * 8 * 4


@pytest.mark.parametrize("change,code", [
    (dict(dtype=7), ARG), (dict(y_rows=-1), ARG), (dict(width=0), ARG), (dict(k=0), ARG), (dict(rows=-1), ARG), (dict(y=None), ARG),
    (dict(slots=None), ARG), (dict(weights=None), ARG), (dict(out=None), ARG), (dict(rows=1 << 31), ARG), (dict(rows=0), 0),
])
def test_expert_combine_refuses(change, code):
    a = dict(y=P, dtype=2, y_rows=20, width=64, slots=P, weights=P, rows=10, k=2, out=P)
    a.update(change)
    rc = _lib.lib().fd_expert_combine(a["y"], a["dtype"], a["y_rows"], a["width"], a["slots"], a["weights"], a["rows"], a["k"], a["out"], None)
    assert rc == code and (rc == 0 or "fd_expert_combine" in _err())


@pytest.mark.parametrize("change,code", [
    (dict(x_dtype=3), ARG), (dict(x_dtype=1, h_dtype=2), ARG), (dict(rows=-1), ARG), (dict(width=0), ARG), (dict(width=16385), LIMIT),
    (dict(x=None), ARG), (dict(x_out=None), ARG), (dict(u=None), ARG), (dict(eps=0.0), ARG), (dict(eps=float("nan")), ARG),
    (dict(gate=P, gate_rows=3), ARG), (dict(gate=P, gate_rows=0), ARG), (dict(gate=P, gate_rows=1, gate_dtype=1), ARG),
    (dict(gate=P, gate_rows=1, gate_act=3), ARG), (dict(post_bias=P), ARG), (dict(pre_bias=P, pre_weight=None), ARG),
    (dict(slots=P), ARG), (dict(slots=P, weights=P, k=0), ARG), (dict(h=None, post_weight=P), ARG), (dict(h=None, pre_weight=None), ARG),
    (dict(rows=1 << 31), ARG), (dict(rows=0), 0),
])
def test_residual_norm_refuses(change, code):
    a = dict(x=P, h=P, x_out=P, u=P, pre_weight=P, rows=10, h_rows=10, width=64, x_dtype=0, h_dtype=0, gate_dtype=0, scale=1.0, eps=1e-6)
    a.update(change)
    args = _lib.NormArgs(**a)
    rc = _lib.lib().fd_residual_norm(C.byref(args), None)
    assert rc == code and (rc == 0 or "fd_residual_norm" in _err())


def test_residual_norm_refuses_no_arguments():
    assert _lib.lib().fd_residual_norm(None, None) == ARG
