"""The expert-block operators (ops.expert_route, expert_linear, expert_combine, block_norm, residual_norm) against their
definitions in float64.

Tolerances, with u = 2^-24 (a float32 rounding) and half a step of the output's type for the one rounding at the end:

* products: a sum of K terms taken in any order is off by at most about K * 2u * sum |x w| where an adder may also cut instead
  of round (2u a step); an activation passes at most 1.13 times that on, and adds some units in the last place of its own;
* norms: a float32 sum of the squares of a row is at most 64 additions deep in a lane and 8 across lanes, the mean of a
  layer norm likewise, so the scale is off by at most 80u and a centred value by 80u of the row's mean magnitude;
* weighted sums: k terms, (k + 1) * u * sum |w y|.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _close(got, want, tol):
    """|got - want| <= tol + half a step of got's type (a subnormal float16 step is 2^-24)."""
    half = want.abs() * (torch.finfo(got.dtype).eps / 2) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    bad = ~((got.double() - want).abs() <= tol * (1 + 2.0 ** -7) + half)
    assert not bool(bad.any()), "%d of %d values off, worst %.3g over its bound" % (
        int(bad.sum()), bad.numel(), float(((got.double() - want).abs() - tol - half).max()))


# ---------------------------------------------------------------------------------------------------------------
# route
def _route64(logits, k, mask, normalize):
    """The definition, in Python on the host: lists of choices, float64 weights."""
    v = logits.double().cpu().numpy()
    T, E = v.shape
    weights, chosen = np.zeros((T, k)), np.full((T, k), -1, np.int32)
    for t in range(T):
        if mask is not None and not mask[t]:
            continue
        ok = [e for e in range(E) if v[t, e] > -math.inf]
        best = sorted(ok, key=lambda e: (-v[t, e], e))[:k]
        if not best:
            continue
        top = v[t, best[0]]
        power = {e: 1.0 if v[t, e] == top else math.exp(v[t, e] - top) for e in ok}
        total = sum(power[e] for e in (best if normalize else ok))
        for j, e in enumerate(best):
            weights[t, j], chosen[t, j] = power[e] / total, e
    slots, rows, offsets = np.full((T, k), -1, np.int32), np.full((T * k,), -1, np.int32), np.zeros((E + 1,), np.int32)
    at = 0
    for e in range(E):
        for t, j in np.argwhere(chosen == e):
            slots[t, j], rows[at] = at, t
            at += 1
        offsets[e + 1] = at
    return weights, chosen, slots, offsets, rows


def _check_route(logits, k, mask=None, normalize=True):
    from facedetection_amd import ops
    r = ops.expert_route(logits, k, mask=mask, normalize=normalize)
    want = _route64(logits, k, None if mask is None else mask.cpu().numpy(), normalize)
    for got, ref, name in zip(r[1:], want[1:], ("experts", "slots", "offsets", "rows")):
        np.testing.assert_array_equal(got.cpu().numpy(), ref, err_msg=name)
    # exp, the sum of up to E of them and the division: a few units each, relative, plus what a difference of logits up to
    # 2^7 loses in float32 (the difference is rounded once, u * 2^7 at most in the exponent)
    tol = (logits.shape[1] + 16) * U + 2.0 ** 7 * U
    np.testing.assert_allclose(r.weights.cpu().numpy(), want[0], rtol=tol, atol=1e-37)
    return r


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,E,k,normalize,masked", [
    (1, 1, 1, True, False), (1, 5, 2, False, False), (10, 8, 2, True, False), (63, 33, 3, False, True), (512, 64, 4, True, True),
    (513, 7, 7, True, False), (700, 200, 5, False, False), (1025, 512, 16, True, True), (2500, 31, 9, False, True), (64, 65, 8, True, False), (64, 300, 16, False, True), (65, 300, 16, False, True), (40, 64, 3, False, False),
])
def test_route(dtype, T, E, k, normalize, masked):
    g = _gen(T * 1000 + E)
    logits = (torch.randn((T, E), generator=g, device="cuda") * 2).to(dtype)         # 16-bit logits tie often
    mask = (torch.rand((T,), generator=g, device="cuda") < 0.7) if masked else None
    _check_route(logits, k, mask, normalize)


@pytest.mark.parametrize("normalize", [True, False])
def test_route_special_logits(normalize):
    inf, nan = math.inf, math.nan
    rows = [
        [0.0, 0.0, 0.0, 0.0, 0.0],                    # all equal: the lowest experts
        [-0.0, 0.0, -0.0, 0.0, 0.0],                  # signed zeros are equal
        [-inf, -inf, -inf, -inf, -inf],               # nothing to choose
        [nan, nan, nan, nan, nan],
        [nan, 1.0, -inf, nan, 0.5],                   # two choices for k = 3
        [inf, 1.0, inf, 0.0, -inf],                   # infinite logits share the weight
        [-3.0e38, -3.3e38, -3.4e38, -3.2e38, -3.1e38],
        [3.4e38, -3.4e38, 0.0, 1.0, 2.0],             # a difference beyond float32
        [1e-45, 0.0, 2e-45, -1e-45, 0.0],             # subnormals
    ]
    logits = torch.tensor(rows * 70, dtype=torch.float32, device="cuda")     # 630 rows: more than one workgroup
    _check_route(logits[:9].contiguous(), 3, None, normalize)
    _check_route(logits, 3, None, normalize)


def test_route_everyone_to_one_expert_and_nobody():
    from facedetection_amd import ops
    logits = torch.zeros((3000, 16), device="cuda")
    logits[:, 11] = 5.0
    r = _check_route(logits, 1)
    assert r.offsets.tolist() == [0] * 12 + [3000] * 5
    r = _check_route(logits, 2, mask=torch.zeros(3000, dtype=torch.uint8, device="cuda"))
    assert r.offsets.tolist() == [0] * 17 and bool((r.rows == -1).all()) and bool((r.weights == 0).all())
    r = ops.expert_route(torch.empty((0, 16), device="cuda"), 2)
    assert r.offsets.tolist() == [0] * 17 and r.rows.numel() == 0 and r.slots.shape == (0, 2)


def test_route_takes_views_and_numpy():
    from facedetection_amd import ops
    wide = torch.randn((40, 24), generator=_gen(5), device="cuda")
    a = ops.expert_route(wide[:, 3:20], 4)
    b = ops.expert_route(wide[:, 3:20].contiguous(), 4)
    c = ops.expert_route(wide[:, 3:20].cpu().numpy(), 4)
    d = ops.expert_route(wide.reshape(-1)[1:86].reshape(5, 17), 4)         # rows that start off a 16-byte border
    for p, q, n in zip(a, b, c):
        assert torch.equal(p, q)
        np.testing.assert_array_equal(p.cpu().numpy(), n)
    _check_route(wide.reshape(-1)[1:86].reshape(5, 17), 4)
    assert d.experts.shape == (5, 4)


# ---------------------------------------------------------------------------------------------------------------
# products
def _act64(v, name):
    if name == "relu":
        return v.clamp(min=0)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v * math.sqrt(0.5))
    return v


def _linear64(x, w, offsets, rows, bias, act, gated):
    """(values, error bound) of the definition."""
    S = x.shape[0] if rows is None else rows.numel()
    E, n, K = w.shape
    N = n // 2 if gated else n
    y, tol = torch.zeros((S, N), dtype=torch.float64, device="cuda"), torch.zeros((S, N), dtype=torch.float64, device="cuda")
    off = offsets.tolist()
    for e in range(E):
        lo, hi = off[e], off[e + 1]
        if lo == hi:
            continue
        xs = x[lo:hi].double() if rows is None else x[rows[lo:hi].long().clamp(min=0)].double() * (rows[lo:hi] >= 0)[:, None]
        we = w[e].double()
        v = xs @ we.t().contiguous()
        t = 2 * (K + 2) * U * (xs.abs() @ we.abs().t().contiguous())
        if bias is not None:
            v, t = v + bias[e].double(), t + 2 * U * bias[e].double().abs()
        a = _act64(v[:, :N], act)
        ta = 1.13 * t[:, :N] + 16 * U * a.abs() + (8 * U * v[:, :N].abs() if act else 0.0)
        if gated:
            ta = ta * (v[:, N:].abs() + t[:, N:]) + a.abs() * t[:, N:] + U * (a * v[:, N:]).abs()
            a = a * v[:, N:]
        y[lo:hi], tol[lo:hi] = a, ta
    return y, tol


def _routing(g, T, E, k, skew, drop):
    """(rows, offsets, slots, weights) of a ragged routing made without the operator."""
    share = -skew * torch.log(torch.arange(1, E + 1, device="cuda").float())
    noise = -torch.log(-torch.log(torch.rand((T, E), generator=g, device="cuda").clamp(1e-6, 1 - 1e-6)))
    chosen = (share + noise).topk(k, dim=1).indices
    chosen[torch.rand((T,), generator=g, device="cuda") < drop] = E
    flat = chosen.reshape(-1)
    by, order = torch.sort(flat, stable=True)
    rows = (order // k).int()
    rows[by == E] = -1
    offsets = torch.searchsorted(by, torch.arange(E + 1, device="cuda")).int()
    slots = torch.empty_like(flat)
    slots[order] = torch.arange(flat.numel(), device="cuda")
    slots[flat == E] = -1
    return rows, offsets, slots.reshape(T, k).int(), torch.rand((T, k), generator=g, device="cuda")


# T, k, E, K, N, act, gated, bias, gather, skew, drop: one slot, odd everything, empty experts, one crowded expert, long and short K
LINEAR = [
    (1, 1, 1, 1, 1, None, False, False, True, 0.0, 0.0),
    (1, 2, 3, 7, 5, "relu", False, True, True, 0.0, 0.0),
    (1, 4, 64, 256, 48, "silu", True, False, True, 0.0, 0.0),
    (10, 2, 8, 512, 64, "silu", True, True, True, 0.0, 0.0),
    (10, 1, 1, 640, 33, None, False, True, False, 0.0, 0.0),
    (17, 1, 2, 40, 24, "gelu", True, True, True, 1.0, 0.5),
    (65, 1, 4, 33, 17, "gelu", False, True, True, 1.0, 0.0),
    (130, 3, 11, 129, 97, "silu", True, True, True, 0.5, 0.2),
    (300, 2, 64, 256, 130, None, False, False, True, 2.0, 0.1),
    (1000, 1, 2, 72, 260, "relu", False, True, False, 1.0, 0.0),
    (513, 2, 3, 1000, 136, "silu", True, False, False, 0.5, 0.3),
    (5, 1, 200, 40, 24, None, False, False, True, 0.0, 0.0),
    (700, 4, 5, 64, 512, "gelu", False, False, True, 0.5, 0.05),
    (2100, 1, 7, 320, 64, None, False, True, True, 3.0, 0.0),
    (40, 2, 900, 24, 16, None, False, True, True, 0.0, 0.0),
    (900, 2, 2, 2048, 256, "silu", True, True, True, 0.0, 0.02),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", LINEAR, ids=lambda c: "x".join(str(v) for v in c[:5]))
def test_expert_linear(dtype, case):
    from facedetection_amd import ops
    T, k, E, K, N, act, gated, has_bias, gather, skew, drop = case
    g = _gen(T + 7 * E + K)
    rows, offsets, _, _ = _routing(g, T, E, k, skew, drop)
    n = 2 * N if gated else N
    x = torch.randn((T if gather else T * k, K), generator=g, device="cuda").to(dtype)
    w = (torch.randn((E, n, K), generator=g, device="cuda") / math.sqrt(K)).to(dtype)
    bias = torch.randn((E, n), generator=g, device="cuda").to(dtype) if has_bias else None
    y = ops.expert_linear(x, w, offsets, rows=rows if gather else None, bias=bias, activation=act, gated=gated)
    want, tol = _linear64(x, w, offsets, rows if gather else None, bias, act, gated)
    _close(y, want, tol)
    assert bool((y[int(offsets[-1]):] == 0).all())


def _kernels(call):
    """(result, names of the kernels a call ran)"""
    from facedetection_amd import profiling
    profiling.begin()
    try:
        out = call()
        torch.cuda.synchronize()
    finally:
        rows = profiling.end()
    return out, {r["kernel"] for r in rows}


# large enough for the 256 x 256 tiles: ragged groups, partial tiles in both directions, a partial last step of K, several
# tiles a workgroup, an empty expert; every activation with and without a gate
WIDE = [
    (50000, 2, 3, 200, 1032, "silu", True, True, True, 0.7, 0.1),
    (100000, 1, 3, 264, 2056, None, False, False, True, 0.7, 0.0),
    (100000, 1, 5, 328, 1040, "gelu", False, True, False, 1.0, 0.05),
    (60000, 1, 2, 1000, 1040, "relu", True, False, False, 0.3, 0.0),
    (30000, 4, 10, 512, 768, None, True, True, True, 0.0, 0.02),
    (130560, 1, 1, 264, 2048, "relu", False, True, True, 0.0, 0.01),
    (32000, 2, 4, 320, 1024, "gelu", True, False, True, 2.0, 0.0),
    (65536, 1, 1, 512, 2056, "silu", False, False, False, 0.0, 0.0),
    # 256 and 192 rows a tile where those fill the last round best
    (9496, 1, 1, 136, 1328, "relu", False, True, True, 0.0, 0.0),
    (12228, 1, 1, 200, 600, "silu", True, False, True, 0.0, 0.01),
    (9828, 1, 2, 264, 680, None, True, True, False, 0.2, 0.0),
    (9649, 1, 9, 136, 1464, "gelu", False, True, False, 0.1, 0.0),
    (8444, 1, 1, 136, 480, None, True, True, True, 0.0, 0.0),
    (10660, 1, 1, 136, 840, "gelu", False, False, True, 0.0, 0.0),
    (8157, 1, 1, 264, 616, "relu", True, True, False, 0.0, 0.0),
    (14530, 1, 9, 136, 576, "silu", False, True, True, 0.1, 0.0),
]


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("case", WIDE, ids=lambda c: "x".join(str(v) for v in c[:5]))
def test_expert_linear_largest_tiles(dtype, case):
    from facedetection_amd import ops
    T, k, E, K, N, act, gated, has_bias, gather, skew, drop = case
    g = _gen(T + 7 * E + K)
    rows, offsets, _, _ = _routing(g, T, E, k, skew, drop)
    n = 2 * N if gated else N
    x = torch.randn((T if gather else T * k, K), generator=g, device="cuda").to(dtype)
    w = (torch.randn((E, n, K), generator=g, device="cuda") / math.sqrt(K)).to(dtype)
    bias = torch.randn((E, n), generator=g, device="cuda").to(dtype) if has_bias else None
    y, kernels = _kernels(lambda: ops.expert_linear(x, w, offsets, rows=rows if gather else None, bias=bias, activation=act, gated=gated))
    assert kernels == {"expert_wide"}
    _close(y, *_linear64(x, w, offsets, rows if gather else None, bias, act, gated))
    assert bool((y[int(offsets[-1]):] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_expert_linear_unaligned_views(dtype):
    """x, weight and bias that start one element past a 16-byte border, and x as a slice of wider rows."""
    from facedetection_amd import ops
    g = _gen(11)
    T, E, K, N = 150, 3, 96, 80
    rows, offsets, _, _ = _routing(g, T, E, 2, 0.5, 0.1)
    buf = lambda *s: torch.randn((int(np.prod(s)) + 1,), generator=g, device="cuda").to(dtype)[1:].reshape(s)
    x, w, b = buf(T, K), buf(E, N, K), buf(E, N)
    assert x.data_ptr() % 16 and w.data_ptr() % 16 and x.is_contiguous()
    y = ops.expert_linear(x, w, offsets, rows=rows, bias=b)
    _close(y, *_linear64(x, w, offsets, rows, b, None, False))
    wide = torch.randn((T, 2 * K), generator=g, device="cuda").to(dtype)
    y = ops.expert_linear(wide[:, 5:5 + K], w, offsets, rows=rows)
    _close(y, *_linear64(wide[:, 5:5 + K], w, offsets, rows, None, None, False))


@pytest.mark.parametrize("T,K,N", [(30, 64, 48), (600, 64, 256)])
def test_expert_linear_bad_offsets_and_rows_stay_in_bounds(T, K, N):
    """Offsets that decrease or leave the range are clamped to [the one before, slots]; rows outside x read as zeros."""
    from facedetection_amd import ops
    g = _gen(3)
    x, w = torch.randn((T, K), generator=g, device="cuda"), torch.randn((4, N, K), generator=g, device="cuda")
    offsets = torch.tensor([5, -7, T // 2, 3, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    clamped = torch.tensor([0, 0, T // 2, T // 2, T], dtype=torch.int32, device="cuda")
    rows = torch.arange(T, dtype=torch.int32, device="cuda")
    rows[3], rows[7], rows[T - 1] = -1, T, 2 ** 31 - 1
    good = rows.clone()
    good[3] = good[7] = good[T - 1] = -1
    y = ops.expert_linear(x, w, offsets, rows=rows)
    _close(y, *_linear64(x, w, clamped, good, None, None, False))


def test_expert_linear_rows_do_not_touch_each_other():
    """Infinities and NaN stay in the rows, the experts and the columns they belong to (odd K: the last piece of a row is
    partial and the next row starts behind it)."""
    from facedetection_amd import ops
    g = _gen(4)
    for T, K, N in ((40, 65, 50), (700, 100, 130)):
        for dtype in TYPES:
            rows, offsets, _, _ = _routing(g, T, 3, 1, 0.0, 0.0)
            x = torch.randn((T, K), generator=g, device="cuda").to(dtype)
            w = torch.randn((3, N, K), generator=g, device="cuda").to(dtype)
            clean = ops.expert_linear(x, w, offsets, rows=rows)
            x2, w2 = x.clone(), w.clone()
            x2[9, 0], x2[10, K - 1] = math.nan, math.inf
            w2[1, 17, 0], w2[1, N - 1, K - 1] = math.nan, math.inf
            y = ops.expert_linear(x2, w2, offsets, rows=rows)
            hit = torch.zeros_like(y, dtype=torch.bool)
            hit[(rows == 9) | (rows == 10)] = True
            lo, hi = int(offsets[1]), int(offsets[2])
            hit[lo:hi, 17] = True
            hit[lo:hi, N - 1] = True
            assert torch.equal(y[~hit], clean[~hit])
            assert not bool(torch.isfinite(y[rows == 9]).any())


def test_expert_linear_empty_and_numpy():
    from facedetection_amd import ops
    w = torch.randn((2, 5, 8), device="cuda")
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert ops.expert_linear(torch.empty((0, 8), device="cuda"), w, off).shape == (0, 5)
    rows = torch.full((6,), -1, dtype=torch.int32, device="cuda")
    assert bool((ops.expert_linear(torch.empty((0, 8), device="cuda"), w, off, rows=rows) == 0).all())
    x = torch.randn((4, 8), device="cuda")
    off = torch.tensor([0, 1, 4], dtype=torch.int32, device="cuda")
    a = ops.expert_linear(x, w, off)
    b = ops.expert_linear(x.cpu().numpy(), w.cpu().numpy(), off.cpu().numpy())
    assert isinstance(b, np.ndarray)
    np.testing.assert_array_equal(a.cpu().numpy(), b)


# ---------------------------------------------------------------------------------------------------------------
# weighted sum
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,k,N", [(1, 1, 1), (3, 2, 7), (10, 2, 2048), (77, 8, 33), (500, 3, 1001), (9, 3, 8), (9, 3, 9), (2, 1, 9000), (1300, 4, 64)])
def test_expert_combine(dtype, T, k, N):
    from facedetection_amd import ops
    g = _gen(T + N)
    _, _, slots, weights = _routing(g, T, max(k, 5), k, 0.5, 0.2)
    y = torch.randn((T * k, N), generator=g, device="cuda").to(dtype)
    y[-1] = math.nan                                              # a row that nobody may read: take its slots out
    slots[slots == T * k - 1] = -1
    if T > 2:
        slots[1, 0] = T * k + 5                                   # outside y
    got = ops.expert_combine(y, slots, weights)
    ok = (slots >= 0) & (slots < T * k)
    terms = torch.where(ok[..., None], weights.double()[..., None] * y.double()[slots.clamp(0, T * k - 1).long()], 0.0)
    _close(got, terms.sum(1), (k + 1) * U * terms.abs().sum(1))


# ---------------------------------------------------------------------------------------------------------------
# norms
def _norm64(v, tv, w, b, layer, eps=1e-6):
    """(value, bound) of a norm of v, known to within tv."""
    D = v.shape[1]
    mean = v.mean(1, keepdim=True) if layer else torch.zeros_like(v[:, :1])
    tc = tv + (tv.mean(1, keepdim=True) + 80 * U * v.abs().mean(1, keepdim=True) + U * v.abs() if layer else 0.0)
    c = v - mean
    r = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    # the scale: its own roundings, and half of what the errors of the values put into the mean square
    tr = 80 * U + r * r * (c.abs() * tc + tc * tc).mean(1, keepdim=True)
    out = c * r * w.double()
    tol = (tc * r * (1 + tr) + (c * r).abs() * tr + 4 * U * (c * r).abs()) * w.double().abs()
    if b is not None:
        out = out + b.double()
        tol = tol + U * (out.abs() + b.double().abs())
    return out, tol


NORM_WIDTHS = [1, 3, 4, 5, 7, 8, 9, 33, 64, 128, 129, 256, 257, 511, 512, 771, 1000, 1024, 1025, 2047, 2048, 2500, 4096, 5000, 8192, 9001, 16383, 16384]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", NORM_WIDTHS)
def test_block_norm(dtype, width):
    from facedetection_amd import ops
    g = _gen(width)
    for rows, layer, bias in ((1, False, False), (19, True, True), (2100 if width <= 2048 else 6, width % 2 == 0, True)):
        x = (torch.randn((rows, width), generator=g, device="cuda") * 3 + 1).to(dtype)
        w = 1 + 0.3 * torch.randn((width,), generator=g, device="cuda")
        b = torch.randn((width,), generator=g, device="cuda") if bias else None
        u = ops.block_norm(x, w, b, kind="layer" if layer else "rms")
        assert u.dtype == dtype
        _close(u, *_norm64(x.double(), torch.zeros_like(x, dtype=torch.float64), w, b, layer))


# rows, width, post, pre, layer, gate ("", "row", or the number of gate rows), its activation, k
RESIDUAL = [
    (1, 64, True, True, False, "", None, 0),
    (10, 2048, True, True, False, "row", None, 0),
    (12, 100, True, False, True, 3, "sigmoid", 0),
    (12, 100, False, True, True, 12, "tanh", 0),
    (12, 1000, False, False, False, 1, None, 0),
    (30, 520, True, True, True, 30, "sigmoid", 2),
    (2050, 1024, True, True, False, 2, "sigmoid", 3),
    (2050, 2048, True, True, True, "row", "tanh", 1),
    (9, 4000, True, True, True, 3, None, 2),
    (4, 16384, True, True, True, 2, "sigmoid", 2),
    (300, 40, True, True, False, "", None, 8),
]


@pytest.mark.parametrize("types", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, torch.float16),
                                   (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)], ids=str)
@pytest.mark.parametrize("case", RESIDUAL, ids=str)
def test_residual_norm(types, case):
    from facedetection_amd import ops
    tx, th = types
    T, D, post, pre, layer, gate, act, k = case
    g = _gen(T + D)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    x = (rand(T, D) * 3).to(tx)
    h = rand(T * max(1, k), D).to(th)
    kw = dict(kind="layer" if layer else "rms", scale=0.6, gate_activation=act if gate else None)
    if k:
        _, _, kw["slots"], kw["weights"] = _routing(g, T, max(k, 5), k, 0.3, 0.3)
    for name, on in (("post", post), ("pre", pre)):
        if on:
            kw[name + "_weight"] = 1 + 0.3 * rand(D)
            kw[name + "_bias"] = rand(D) if layer else None
    if gate:
        kw["gate"] = rand(D) if gate == "row" else rand(gate, D).to(th)
    out = ops.residual_norm(x, h, **kw)
    new, u = out if pre else (out, None)
    assert new.dtype == tx and (u is None or u.dtype == th)

    zero = torch.zeros((T, D), dtype=torch.float64, device="cuda")
    if k:
        ok = kw["slots"] >= 0
        terms = torch.where(ok[..., None], kw["weights"].double()[..., None] * h.double()[kw["slots"].clamp(min=0).long()], 0.0)
        v, tv = terms.sum(1), (k + 1) * U * terms.abs().sum(1)
    else:
        v, tv = h.double(), zero
    if post:
        v, tv = _norm64(v, tv, kw["post_weight"], kw.get("post_bias"), layer)
    if gate:
        gv = kw["gate"].double().reshape(-1, D)
        gv = {None: gv, "sigmoid": torch.sigmoid(gv), "tanh": torch.tanh(gv)}[act].repeat_interleave(T // gv.shape[0], 0)
        v, tv = v * gv, tv * gv.abs() + 9 * U * (v * gv).abs()
    scale = float(np.float32(0.6))
    want = x.double() + scale * v
    tol = scale * tv + U * ((scale * v).abs() + want.abs())
    _close(new, want, tol)
    if pre:
        _close(u, *_norm64(want, tol, kw["pre_weight"], kw.get("pre_bias"), layer))


def test_residual_norm_rows_without_a_choice_keep_the_stream():
    from facedetection_amd import ops
    x = torch.randn((6, 256), device="cuda")
    y = torch.full((12, 256), math.nan, device="cuda")
    slots = torch.full((6, 2), -1, dtype=torch.int32, device="cuda")
    new = ops.residual_norm(x, y, post_weight=torch.ones(256, device="cuda"), slots=slots, weights=torch.ones((6, 2), device="cuda"))
    assert torch.equal(new, x)


# ---------------------------------------------------------------------------------------------------------------
# refusals
def test_refusals():
    from facedetection_amd import ops
    x, w = torch.zeros((4, 8), device="cuda"), torch.zeros((2, 6, 8), device="cuda")
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    one, sl, wt = torch.ones(8, device="cuda"), torch.zeros((4, 2), dtype=torch.int32, device="cuda"), torch.zeros((4, 2), device="cuda")
    bad = [
        lambda: ops.expert_route(x[0], 1), lambda: ops.expert_route(x, 0), lambda: ops.expert_route(x, 9),
        lambda: ops.expert_route(x, 1, mask=torch.ones(5, dtype=torch.bool, device="cuda")),
        lambda: ops.expert_route(x, 1, mask=torch.ones(4, device="cuda")),
        lambda: ops.expert_linear(x[0], w, off), lambda: ops.expert_linear(x, w[0], off), lambda: ops.expert_linear(x, w[:, :, :7], off),
        lambda: ops.expert_linear(x, w.half(), off), lambda: ops.expert_linear(x, w, off[:2]), lambda: ops.expert_linear(x, w, off.long()),
        lambda: ops.expert_linear(x, w, off, rows=torch.zeros(4, dtype=torch.int64, device="cuda")),
        lambda: ops.expert_linear(x, w, off, rows=sl), lambda: ops.expert_linear(x, w, off, bias=torch.zeros(6, device="cuda")),
        lambda: ops.expert_linear(x, w, off, bias=torch.zeros((2, 6), device="cuda", dtype=torch.bfloat16)),
        lambda: ops.expert_linear(x, w, off, activation="swish"), lambda: ops.expert_linear(x, w[:, :5], off, gated=True),
        lambda: ops.expert_combine(x, sl, wt[:, :1]), lambda: ops.expert_combine(x, sl.long(), wt),
        lambda: ops.expert_combine(x[0], sl, wt), lambda: ops.expert_combine(x, sl[:, :0], wt[:, :0]),
        lambda: ops.block_norm(x, one[:7]), lambda: ops.block_norm(x[0], one), lambda: ops.block_norm(x, one, kind="batch"),
        lambda: ops.residual_norm(x, x[:3]), lambda: ops.residual_norm(x, x[:, :7]), lambda: ops.residual_norm(x.half(), x),
        lambda: ops.residual_norm(x.half(), x.bfloat16()), lambda: ops.residual_norm(x, x, gate=one[:7]),
        lambda: ops.residual_norm(x, x, gate=torch.ones((3, 8), device="cuda")), lambda: ops.residual_norm(x, x, gate=one, gate_activation="relu"),
        lambda: ops.residual_norm(x, x, gate_activation="tanh"), lambda: ops.residual_norm(x, x, post_bias=one),
        lambda: ops.residual_norm(x, x, slots=sl), lambda: ops.residual_norm(x, x, slots=sl[:3], weights=wt[:3]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was accepted" % i)
    from facedetection_amd._lib import FaceDetError
    for call in (lambda: ops.block_norm(torch.zeros((2, 16385), device="cuda"), torch.ones(16385, device="cuda")),
                 lambda: ops.block_norm(x, one, eps=0.0),
                 lambda: ops.expert_route(torch.zeros((2, 513), device="cuda"), 1),
                 lambda: ops.expert_linear(x, torch.zeros((1025, 1, 8), device="cuda"), torch.zeros(1026, dtype=torch.int32, device="cuda"))):
        with pytest.raises(FaceDetError):
            call()


# ---------------------------------------------------------------------------------------------------------------
# the operators together, as a block of a network runs
def _block(x, u, p):
    """One expert block: route, gated product, product, expert sum + norm + gate + residual + next norm."""
    from facedetection_amd import ops
    r = ops.expert_route(ops.expert_linear(u, p["router"][None], p["all"]), 2)       # one expert: the router's product
    a = ops.expert_linear(u, p["up"], r.offsets, rows=r.rows, activation="silu", gated=True)
    y = ops.expert_linear(a, p["down"], r.offsets)
    return r, y, ops.residual_norm(x, y, post_weight=p["post"], gate=p["gate"], gate_activation="sigmoid", scale=0.5, pre_weight=p["pre"],
                                   slots=r.slots, weights=r.weights)


def _block_params(g, T, D, F, E, frames, dtype):
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")
    return dict(all=torch.tensor([0, T], dtype=torch.int32, device="cuda"), router=(rand(E, D) / math.sqrt(D)).to(dtype), up=(rand(E, 2 * F, D) / math.sqrt(D)).to(dtype),
                down=(rand(E, D, F) / math.sqrt(F)).to(dtype), post=1 + 0.1 * rand(D), pre=1 + 0.1 * rand(D), gate=rand(frames, D))


@pytest.mark.parametrize("T,frames", [(10, 1), (160, 16), (1, 1), (1200, 3)])
def test_expert_block_end_to_end(T, frames):
    """float32 throughout against float64 with the operator's own choices (a near tie may fall either way)."""
    g = _gen(T)
    D, F, E = 96, 72, 6
    p = _block_params(g, T, D, F, E, frames, torch.float32)
    from facedetection_amd import ops
    x = torch.randn((T, D), generator=g, device="cuda")
    u = ops.block_norm(x, p["pre"])
    r, y, (new, nxt) = _block(x, u, p)
    rms = lambda v, w: v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6) * w.double()
    u64 = rms(x.double(), p["pre"])
    logits = u64 @ p["router"].double().t().contiguous()
    h = torch.zeros_like(u64)
    wts = torch.softmax(logits.gather(1, r.experts.long()), 1)
    for j in range(2):
        for e in range(E):
            sel = r.experts[:, j] == e
            v = u64[sel] @ p["up"][e].double().t().contiguous()
            h[sel] += wts[sel, j:j + 1] * ((torch.nn.functional.silu(v[:, :F]) * v[:, F:]) @ p["down"][e].double().t().contiguous())
    best = logits.topk(3, dim=1).values
    assert bool((logits.gather(1, r.experts.long()).sort(1, descending=True).values >= best[:, :2] - 1e-5).all())
    want = x.double() + 0.5 * torch.sigmoid(p["gate"].double()).repeat_interleave(T // frames, 0) * rms(h, p["post"])
    # float32 all the way: products of 96 and 72 terms, three norms; 2^-24 * (2 * 96 + 2 * 72 + 3 * 80) times values of order 1,
    # which the norm after the block may scale up by 1 / rms(h)
    scale = float((1.0 / h.pow(2).mean(1).sqrt()).max().clamp(min=1.0))
    tol = 576 * U * 4 * scale
    assert float((new.double() - want).abs().max()) <= tol * float(want.abs().max())
    assert float((nxt.double() - rms(want, p["pre"])).abs().max()) <= 2 * tol * float(want.abs().max())


def test_expert_block_in_a_graph_and_on_another_stream():
    """Captured on a side stream and replayed with new input, with eager work between the replays."""
    from facedetection_amd import ops
    g = _gen(77)
    T, D, F, E = 200, 256, 128, 8
    p = _block_params(g, T, D, F, E, 4, torch.bfloat16)
    xs = [torch.randn((T, D), generator=g, device="cuda") for _ in range(3)]
    buf = xs[0].clone()

    def step(x):
        u = ops.block_norm(x.bfloat16(), p["pre"])
        _, y, (new, nxt) = _block(x, u, p)
        return y, new, nxt

    want = [[t.clone() for t in step(x)] for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(xs[1])
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want[1]):
        assert torch.equal(a, b)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buf)
    with torch.cuda.graph(other):
        out2 = step(xs[2])
    for i in (0, 1, 2, 1, 0):
        buf.copy_(xs[i])
        graph.replay()
        other.replay()
        eager = step(xs[(i + 1) % 3])
        torch.cuda.synchronize()
        for a, b, c, d, e in zip(out, want[i], out2, want[2], eager):
            assert torch.equal(a, b) and torch.equal(c, d)
        for a, b in zip(eager, want[(i + 1) % 3]):
            assert torch.equal(a, b)


def test_same_bits_every_time():
    from facedetection_amd import ops
    g = _gen(9)
    logits = torch.randn((4000, 32), generator=g, device="cuda")
    x = torch.randn((4000, 128), generator=g, device="cuda").bfloat16()
    w = torch.randn((32, 192, 128), generator=g, device="cuda").bfloat16()
    first = None
    for _ in range(5):
        r = ops.expert_route(logits, 4)
        y = ops.expert_linear(x, w, r.offsets, rows=r.rows)
        out = list(r) + [y, ops.expert_combine(y, r.slots, r.weights)]
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(out, first))
        first = out


# ---------------------------------------------------------------------------------------------------------------
# more than 2^31 bytes, elements or threads, and values that are no numbers
def test_block_norm_of_more_rows_than_a_grid_dimension_has_threads():
    from facedetection_amd import ops
    T = 2 ** 28 + 5                                            # 16 lanes a row: 2^32 threads and some
    x = torch.ones((T, 1), dtype=torch.float16, device="cuda")
    x[-3:, 0] = torch.tensor([0.0, -3.0, 0.5], device="cuda")
    x[2 ** 27 - 1:2 ** 27 + 2, 0] = -2.0
    u = ops.block_norm(x, torch.full((1,), 2.0, device="cuda"), bias=torch.full((1,), 1.0, device="cuda"))
    # x / sqrt(x^2 + 1e-6) is 1 to 2e-6 (at 0.5): 3, -1 and 1, to half a step of float16 behind it
    want = 1.0 + 2.0 * torch.sign(x)
    assert float((u - want).abs().max()) <= 2.0 ** -9


def test_expert_combine_of_more_rows_than_a_grid_dimension_has_threads():
    from facedetection_amd import ops
    if torch.cuda.mem_get_info()[0] < 100 * 2 ** 30:
        pytest.skip("an output of 64 GiB")
    T, N = 2 ** 24 + 3, 2048                                   # a workgroup of 256 a row
    y = torch.randn((4, N), generator=_gen(1), device="cuda").half()
    slots = (torch.arange(T, dtype=torch.int32, device="cuda") % 5 - 1)[:, None].contiguous()
    out = ops.expert_combine(y, slots, torch.full((T, 1), 0.5, device="cuda"))
    for at in (0, 2 ** 23 - 2, T - 6):
        want = torch.where(slots[at:at + 6] >= 0, 0.5 * y[slots[at:at + 6, 0].long().clamp(min=0)].float(), 0.0).half()
        assert torch.equal(out[at:at + 6], want)
    del out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("T,E,k,masked", [(262144, 9, 2, True), (262145, 9, 2, False), (300001, 100, 4, True), (270000, 512, 3, False), (1300000, 2, 1, True),
                                          (700003, 17, 9, False)])
def test_route_of_many_rows(T, E, k, masked):
    """Several hundred workgroups and more, whose counts are joined another way, against stable sorts."""
    from facedetection_amd import ops
    g = _gen(T + E)
    logits = torch.randn((T, E), generator=g, device="cuda")
    mask = torch.rand((T,), generator=g, device="cuda") < 0.6 if masked else None
    r = ops.expert_route(logits, k, mask=mask)
    by, chosen = logits.sort(dim=1, descending=True, stable=True)
    weights, chosen = torch.softmax(by[:, :k].double(), 1), chosen[:, :k].int()
    if masked:
        weights, chosen = weights * mask[:, None], torch.where(mask[:, None], chosen, -1)
    assert torch.equal(r.experts, chosen)
    assert float((r.weights - weights).abs().max()) <= (k + 16 + 2.0 ** 7) * U
    flat = torch.where(chosen < 0, E, chosen).reshape(-1)
    by, order = flat.sort(stable=True)
    assert torch.equal(r.offsets, torch.searchsorted(by, torch.arange(E + 1, dtype=torch.int32, device="cuda")).int())
    n = int(r.offsets[-1])
    assert torch.equal(r.rows[:n], (order[:n] // k).int()) and bool((r.rows[n:] == -1).all())
    slots = torch.full_like(flat, -1)
    slots[order[:n]] = torch.arange(n, dtype=torch.int32, device="cuda")
    assert torch.equal(r.slots.reshape(-1), slots)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,E,k,normalize,masked", [
    (17, 8, 2, True, False), (300, 31, 4, False, True), (512, 8, 1, True, True), (513, 12, 2, False, False), (400, 15, 8, True, False),
    (505, 30, 16, False, True), (8200, 17, 5, True, True), (17, 32, 3, True, False), (16, 512, 16, False, False), (8192, 16, 2, False, True),
    (2500, 257, 4, True, False), (1100, 450, 7, False, True), (300, 1, 1, True, True), (4000, 6, 6, False, False)])
def test_route_at_the_borders_of_its_kernels(dtype, T, E, k, normalize, masked):
    test_route(dtype, T, E, k, normalize, masked)


@pytest.mark.parametrize("dtype,bits,quiet", [(torch.float32, torch.int32, 0x7f800001), (torch.float16, torch.int16, 0x7c01),
                                              (torch.bfloat16, torch.int16, 0x7f81)])
@pytest.mark.parametrize("T", [40, 700])
def test_route_signalling_nan_is_not_chosen(dtype, bits, quiet, T):
    logits = torch.randn((T, 12), generator=_gen(T), device="cuda").to(dtype)
    logits.view(bits)[::3, 4] = quiet
    logits.view(bits)[1::7, :11] = quiet
    assert int(torch.isnan(logits).sum()) > T // 3
    for normalize in (True, False):
        _check_route(logits, 3, None, normalize)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,K,N", [(3, 40, 24), (500, 40, 72), (3000, 256, 256), (3000, 251, 129), (66000, 192, 2048)])
def test_expert_linear_nan_passes_every_activation(dtype, T, K, N):
    from facedetection_amd import ops
    g = _gen(T)
    x, w = torch.randn((T, K), generator=g, device="cuda").to(dtype), torch.randn((1, 2 * N, K), generator=g, device="cuda").to(dtype)
    off = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    x[T // 2, K // 3] = math.nan
    for act in (None, "relu", "silu", "gelu"):
        for gated in (False, True):
            y = ops.expert_linear(x, w, off, activation=act, gated=gated)
            bad = torch.isnan(y)
            assert bool(bad[T // 2].all()) and int(bad.sum()) == y.shape[1]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,N", [(3, 40), (700, 200), (50000, 1024)])
def test_expert_linear_of_no_rows_at_all(dtype, S, N):
    """x has no rows: every index lies outside of it, and a slot of an expert is the activation of its bias."""
    from facedetection_amd import ops
    g = _gen(S)
    w, b = torch.randn((2, N, 512), generator=g, device="cuda").to(dtype), torch.randn((2, N), generator=g, device="cuda").to(dtype)
    off = torch.tensor([0, S // 3, S - 1], dtype=torch.int32, device="cuda")
    rows = torch.arange(S, dtype=torch.int32, device="cuda") - 1
    y = ops.expert_linear(torch.empty((0, 512), dtype=dtype, device="cuda"), w, off, rows=rows, bias=b, activation="relu")
    want = torch.cat([b[0].relu().expand(S // 3, N), b[1].relu().expand(S - 1 - S // 3, N), torch.zeros((1, N), dtype=dtype, device="cuda")])
    assert torch.equal(y, want)


@pytest.mark.parametrize("K,N,S,gather,per", [
    (1024, 64, 2 ** 22 + 77, False, 1), (1024, 64, 3000, True, 1), (1021, 64, 3000, True, 1), (1024, 1024, 40000, True, 1),
    (64, 1024, 2 ** 21 + 300, False, 1), (8, 1000, 2 ** 22 + 9, False, 1), (1024, 24, 5, True, 1), (512, 512, 2 ** 22 + 500, False, 2)])
def test_expert_linear_beyond_31_bits(K, N, S, gather, per):
    """x or y of more than 2^31 bytes or elements: slots at both ends and in the middle, rows at the end of x."""
    from facedetection_amd import ops
    g = _gen(K + N)
    T = 2 ** 22 + 1234 if gather else S
    x = torch.empty((T, K), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w = (torch.randn((per, N, K), generator=g, device="cuda") / math.sqrt(K)).bfloat16()
    bias = torch.randn((per, N), generator=g, device="cuda").bfloat16()
    rows = None
    if gather:
        rows = (T - 1 - torch.randint(0, T, (S,), generator=g, device="cuda") // 3).int()
        rows[0], rows[S // 2], rows[-2] = 0, T - 1, T
    bound = torch.tensor([0] + [(S - 1) * (e + 1) // per for e in range(per)], dtype=torch.int32, device="cuda")
    y = ops.expert_linear(x, w, bound, rows=rows, bias=bias)
    assert y.shape == (S, N) and bool((y[-1] == 0).all())
    pick = torch.cat([torch.arange(0, min(S, 300)), torch.arange(S // 2 - min(S // 2, 150), S // 2 + min(S // 2, 150)),
                      torch.arange(max(0, S - 300), S - 1)]).unique().cuda()
    src = pick if rows is None else rows[pick].long()
    xs = torch.where((src < T)[:, None], x[src.clamp(max=T - 1)], 0.0)
    at = torch.searchsorted(pick, bound[1:].long()).int()
    _close(y[pick], *_linear64(xs, w, torch.cat([torch.zeros_like(at[:1]), at]), None, bias, None, False))


# more kinds of tiles: one row list entry more or less than a tile, more than 64 experts, two and three steps of K, and the
# widths at which another tile is the cheaper one
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [
    (8000, 2, 70, 512, 264, "silu", True, True, True, 0.3, 0.1), (20000, 2, 130, 192, 520, None, False, True, True, 0.3, 0.02),
    (3000, 2, 16, 128, 512, "silu", True, False, True, 0.3, 0.0), (12000, 1, 8, 512, 2048, None, False, True, True, 0.1, 0.0),
    (4000, 2, 32, 1024, 1024, "silu", True, False, True, 0.5, 0.0), (600, 2, 16, 512, 512, "gelu", False, False, False, 0.5, 0.1),
    (398, 2, 50, 416, 1003, "relu", False, True, True, 0.5, 0.0), (64, 1, 1, 2048, 256, None, False, True, True, 0.0, 0.0),
    (20, 2, 2, 4104, 100, "silu", True, True, True, 0.0, 0.0), (3000, 1, 4, 1001, 300, None, False, False, True, 0.5, 0.0),
    (17532, 1, 20, 72, 136, "silu", True, True, True, 0.1, 0.0), (9838, 1, 20, 72, 131, None, True, False, False, 0.1, 0.0),
    (13750, 2, 9, 72, 83, "relu", True, True, True, 0.1, 0.02), (30000, 1, 5, 73, 150, "gelu", True, True, True, 0.1, 0.0),
    (5229, 1, 2, 72, 38, "silu", True, False, True, 0.1, 0.0), (200, 1, 1, 1024, 256, "silu", False, True, True, 0.0, 0.0),
    (500, 1, 1, 2048, 256, "gelu", True, True, False, 0.0, 0.01), (158, 2, 2, 1215, 768, "silu", False, False, True, 1.0, 0.2),
    (100, 1, 1, 4104, 40, None, True, False, True, 0.0, 0.0), (333, 3, 4, 515, 77, "relu", True, True, True, 0.5, 0.1), (30000, 2, 2, 249, 448, "gelu", False, True, True, 0.5, 0.0), (257, 1, 1, 192, 520, None, True, False, True, 0.0, 0.0),
], ids=lambda c: "x".join(str(v) for v in c[:5]))
def test_expert_linear_other_tiles(dtype, case):
    test_expert_linear(dtype, case)
