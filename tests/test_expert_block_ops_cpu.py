"""Argument checks of the expert-block operators in ops.py that come before anything is moved to the GPU.  Sizes that a C int
does not hold would reach the library as other sizes.  No GPU work: the tensors are one element seen many times."""
import pytest
import torch

from facedetection_amd import _lib, ops, runtime

WIDE = 2 ** 32 + 64          # 64 in an int


@pytest.fixture(autouse=True)
def no_gpu(monkeypatch):
    monkeypatch.setattr(runtime, "current", lambda: (0, 0))
    monkeypatch.setattr(runtime, "rows_to_device", lambda array, dtype, index: array)


def _seen(*shape, dtype=torch.float16):
    return torch.zeros((), dtype=dtype).expand(shape)


@pytest.mark.parametrize("width", [2 ** 31, WIDE])
def test_widths_beyond_an_int_are_refused(width):
    x, one, sl, wt = _seen(1, width), _seen(width, dtype=torch.float32), _seen(1, 2, dtype=torch.int32), _seen(1, 2, dtype=torch.float32)
    off = _seen(2, dtype=torch.int32)
    calls = [
        lambda: ops.expert_route(x, 1),
        lambda: ops.expert_linear(x, _seen(1, 8, width), off),
        lambda: ops.expert_linear(_seen(1, 8), _seen(1, width, 8), off),
        lambda: ops.expert_linear(_seen(1, 8), _seen(width, 1, 8), _seen(width + 1, dtype=torch.int32)),
        lambda: ops.expert_combine(x, sl, wt),
        lambda: ops.expert_combine(_seen(1, 8), _seen(1, width, dtype=torch.int32), _seen(1, width, dtype=torch.float32)),
        lambda: ops.block_norm(x, one),
        lambda: ops.residual_norm(x, x),
        lambda: ops.residual_norm(_seen(1, 8), _seen(1, 8), slots=_seen(1, width, dtype=torch.int32), weights=_seen(1, width, dtype=torch.float32)),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="at most 2147483647"):
            call()
            pytest.fail("call %d was accepted" % i)


@pytest.mark.parametrize("change", [dict(dtype=3), dict(inner=0), dict(outputs=0), dict(rows=None, slots=9), dict(experts=1025), dict(slots=(1 << 31) - 1024)])
def test_expert_linear_kernel_names_a_kernel_for_what_the_operator_takes(change):
    L = _lib.lib()
    a = dict(x=4096, dtype=2, x_rows=8, inner=64, weight=4096, experts=4, outputs=8, rows=4096, slots=16, gated=0)
    assert L.fd_expert_linear_kernel(*a.values()) == b"stream 16 rows, 4 waves"
    assert L.fd_expert_linear_kernel(*dict(a, slots=0).values()) == b""
    a.update(change)
    assert L.fd_expert_linear_kernel(*a.values()) is None and b"fd_expert_linear" in L.fd_last_error()


def test_expert_linear_of_an_empty_row_list():
    """An empty list has no address; it is no call without a list, whose rows would all be slots."""
    y = ops.expert_linear(torch.ones((4, 8)), torch.ones((2, 5, 8)), torch.zeros(3, dtype=torch.int32), rows=torch.zeros(0, dtype=torch.int32))
    assert y.shape == (0, 5)
