"""The expert-block operators at the ends of what their documentation allows, against float64 or exact results."""
import math

import numpy as np
import pytest
import torch

from test_gpu_expert_block import TYPES, U, _close, _gen, _norm64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N", [2 ** 31 - 1, 2 ** 31 - 2 ** 27 + 9])
def test_expert_combine_of_the_widest_rows(N):
    """Columns up to the last that an int counts: half of a float16 is exact down to 2^-14, one rounding below."""
    from facedetection_amd import ops
    y = torch.randn((1, N), generator=_gen(2), device="cuda", dtype=torch.float16)
    out = ops.expert_combine(y, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.full((1, 1), 0.5, device="cuda"))
    for lo in range(0, N, 2 ** 28):
        hi = min(N, lo + 2 ** 28)
        assert torch.equal(out[:, lo:hi], y[:, lo:hi] * 0.5)
    del out, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES)
def test_residual_norm_of_no_expert_rows(dtype):
    """h has no rows: no slot adds anything, so the norm after the block is that of zeros, its bias."""
    from facedetection_amd import ops
    g = _gen(3)
    x, bias, gate = torch.randn((7, 100), generator=g, device="cuda"), torch.randn((100,), generator=g, device="cuda"), torch.randn((100,), generator=g, device="cuda")
    slots, weights = torch.arange(14, dtype=torch.int32, device="cuda").reshape(7, 2), torch.ones((7, 2), device="cuda")
    one = torch.ones(100, device="cuda")
    empty = torch.empty((0, 100), dtype=dtype, device="cuda")
    assert torch.equal(ops.residual_norm(x, empty, slots=slots, weights=weights), x)
    new, u = ops.residual_norm(x, empty, slots=slots, weights=weights, post_weight=one, post_bias=bias, gate=gate, scale=0.5, pre_weight=one)
    want = x.double() + 0.5 * (gate.double() * bias.double())
    _close(new, want, 4 * U * (x.double().abs() + want.abs()))
    assert u.dtype == dtype and torch.equal(u, ops.residual_norm(new, torch.zeros((7, 100), dtype=dtype, device="cuda"), pre_weight=one)[1])


def test_expert_block_of_an_empty_batch():
    """No rows at all, with a gate row for each of them and with frames of no rows."""
    from facedetection_amd import ops
    x, one = torch.empty((0, 24), device="cuda"), torch.ones(24, device="cuda")
    r = ops.expert_route(torch.empty((0, 3), device="cuda"), 2)
    u = ops.block_norm(x, one)
    y = ops.expert_linear(u, torch.ones((3, 24, 24), device="cuda"), r.offsets, rows=r.rows)
    assert u.shape == y.shape == (0, 24) and ops.expert_combine(y, r.slots, r.weights).shape == (0, 24)
    for gate in (one, torch.empty((0, 24), device="cuda"), torch.ones((4, 24), device="cuda")):
        for more in ({}, dict(slots=r.slots, weights=r.weights)):
            new, u = ops.residual_norm(x, y, gate=gate, gate_activation="sigmoid", post_weight=one, pre_weight=one, **more)
            assert new.shape == u.shape == (0, 24)


# S, K, N: the stream kernel, the tiles through registers, the tiles by DMA, the large tiles
VALUES = [(3, 1, 1), (4000, 1, 1), (4000, 136, 24), (50000, 136, 1024)]


def _activated(v, S, K, N, act):
    """act of the values v, as products: x has one of them a row and zeros, all weights are one."""
    from facedetection_amd import ops
    x = torch.zeros((S, K), dtype=v.dtype, device="cuda")
    x[:, K // 2] = v[:S] if v.numel() >= S else v.repeat(-(-S // v.numel()))[:S]
    off = torch.tensor([0, S], dtype=torch.int32, device="cuda")
    y = ops.expert_linear(x, torch.ones((1, N, K), dtype=v.dtype, device="cuda"), off, activation=act)
    assert torch.equal(y, y[:, :1].expand(S, N))
    return x[:, K // 2].double(), y[:, 0]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,K,N", VALUES)
def test_gelu_is_good_relative_to_its_value(dtype, S, K, N):
    """The products are exact.  Of the value's own size: for 16 bits the fitted erfc 15 U, its terms, which cancel by less than
    half, 24 U, exp2, factors and the rounding before them 8 U, and the argument v^2 / 2, rounded twice with a rounded constant,
    1.25 v^2 U; for float32 erfcf 32 U, and its argument, rounded once with a rounded constant, 1.3 v^2 U."""
    v = torch.linspace(-12, 12, 4001, device="cuda").to(dtype)
    v = torch.cat([torch.tensor([-6.0, -8.0, 2.0], device="cuda").to(dtype), v])
    v, y = _activated(v, S, K, N, "gelu")
    want = 0.5 * v * torch.special.erfc(-v * math.sqrt(0.5))
    _close(y, want, (48 + 1.5 * v * v) * U * want.abs())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,K,N", VALUES)
def test_silu_is_good_relative_to_its_value(dtype, S, K, N):
    """The products are exact.  float32: exp 6 U, 1 + exp, the factor and the quotient 2 U each at most.  16 bits: the argument of
    exp2, rounded once with a rounded constant, 1.3 |v| U, exp2 and the reciprocal 2 U each, three roundings.  A float32 exp
    below 2^-126 is zero, and so is the result, below 100 * 2^-126."""
    v = torch.linspace(-100, 100, 4001, device="cuda").to(dtype)
    v = torch.cat([torch.tensor([-20.0, -87.5, 8.1], device="cuda").to(dtype), v])
    v, y = _activated(v, S, K, N, "silu")
    want = v * torch.sigmoid(v)
    _close(y, want, (12 if dtype == torch.float32 else 8 + 1.5 * v.abs()) * U * want.abs() + torch.where(v < -87.3, 100 * 2.0 ** -126, 0.0))


@pytest.mark.parametrize("act", ["sigmoid", "tanh"])
@pytest.mark.parametrize("width", [1, 7, 4001])
def test_gate_is_good_relative_to_its_value(act, width):
    """x' = 0 + 1 * act(gate) * 1.  Sigmoid: exp 6 U, 1 + exp, the reciprocal and the factor 2 U each at most; tanhf has 2 units."""
    from facedetection_amd import ops
    g = torch.linspace(-100, 100, 4001, device="cuda")[:, None] if width < 4001 else torch.linspace(-100, 100, 4001, device="cuda")[None]
    gate = g.expand(-1, width).contiguous()
    y = ops.residual_norm(torch.zeros_like(gate), torch.ones_like(gate), gate=gate, gate_activation=act)
    want = torch.sigmoid(gate.double()) if act == "sigmoid" else torch.tanh(gate.double())
    _close(y, want, 12 * U * want.abs() + torch.where((gate < -87.3) & (act == "sigmoid"), 2.0 ** -126, 0.0))
    if act == "sigmoid":
        assert bool((y[gate > -87.3] > 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 7, 250, 400, 1000, 2000, 5000, 16384])
def test_block_norm_of_a_float32_stream(dtype, width):
    """u in a 16-bit type from float32 rows, rounded once: the rows have values that 16 bits do not hold."""
    from facedetection_amd import ops
    g = _gen(width)
    for rows, layer in ((3, True), (2100 if width <= 2048 else 5, False)):
        x = torch.randn((rows, width), generator=g, device="cuda") * 3 + 1000
        w, b = 1 + 0.3 * torch.randn((width,), generator=g, device="cuda"), torch.randn((width,), generator=g, device="cuda")
        u = ops.block_norm(x, w, b if layer else None, kind="layer" if layer else "rms", dtype=dtype)
        assert u.dtype == dtype and u.shape == x.shape
        _close(u, *_norm64(x.double(), torch.zeros_like(x, dtype=torch.float64), w, b if layer else None, layer))


def test_block_norm_refuses_types():
    from facedetection_amd import ops
    x, one = torch.zeros((4, 8), device="cuda"), torch.ones(8, device="cuda")
    assert ops.block_norm(np.ones((4, 8), np.float32), one, dtype=torch.float16).dtype == np.float16
    for call in (lambda: ops.block_norm(x, one, dtype=torch.float64), lambda: ops.block_norm(x.half(), one, dtype=torch.float32),
                 lambda: ops.block_norm(x.half(), one, dtype=torch.bfloat16), lambda: ops.block_norm(x, one, dtype="bfloat16"),
                 lambda: ops.block_norm(np.ones((4, 8), np.float32), one, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("E,k", [(64, 4), (512, 8)])
def test_route_sums_of_all_experts_do_not_gather_roundings(E, k):
    """Softmax over all experts by the kernel that walks a row: the error as a root mean square.  A rounding has 0.41 U (uniform
    over half a step, averaged over the mantissa).  64 experts: the last roundings of the sum 0.6 U together, exp 0.6 U, the quotient
    0.4 U, so 0.9 U.  512: the running sum of 16 parts in each half 0.7 U and the rest as before, so 1.1 U.  A third is left as
    room.  One by one, 32 and 256 terms would be 1.4 U and 2.7 U in the sum alone."""
    from facedetection_amd import ops
    logits = torch.randn((40000 if E == 64 else 70000, E), generator=_gen(E), device="cuda") * 1.5
    r = ops.expert_route(logits, k, normalize=False)
    want = torch.softmax(logits.double(), 1).gather(1, r.experts.long())
    assert float((r.weights.double() - want).norm() / want.norm()) <= (1.2 if E == 64 else 1.5) * U
